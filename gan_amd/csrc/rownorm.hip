// Layer norm over the rows of a dense (rows, D) matrix (gfx950): forward, backward with the reduction of the weight's and
// the bias's gradient, and the backward of the backward (gradient penalties).  For one row, with m = mean x,
// r = (mean (x - m)^2 + eps)^-1/2, t = (x - m) r and P(u) = u - mean u - t mean(u t):
//   forward   y  = t w + b
//   backward  h  = g w;  gx = r P(h);  gw = sum_rows g t;  gb = sum_rows g
//   second    for cotangents v of gx, cw of gw, cb of gb (P is symmetric, dt/dx = r P, dr/dx = -r^2 t / D):
//             gg  = w r P(v) + cw t + cb
//             gxx = r P(g cw - r (v mean(h t) + h mean(v t))) - r^2 t (mean(v h) - mean v mean h - mean(v t) mean(h t))
//             gww = sum_rows g r P(v)
// All three move a few bytes per flop: HBM bounds them.  Each row is read once and kept in registers, 16 bytes a lane and
// load, between its statistics and its results; a row belongs to TPR threads (16 and more) with one or two
// such vectors each (up to 1024 and four in the widest), so that short rows need no LDS and registers leave room for many waves.
// Longer rows are cut into pieces that first sum and then, in a second launch, join the sums and write.
// Column sums: where a workgroup walks over many rows, its threads keep their columns' sums in registers and write one
// partial row per workgroup (fold_cols_k adds those in a fixed order: no atomics, the same bits on every run); where there
// are few rows for that, a second kernel (backward: more workgroups of the same) goes down the columns.
// Sums and statistics are fp32 throughout; bf16 results are rounded once, on the store.
// Measured, launches alone, of 5.0 TB/s that a copy reaches (in brackets the bytes' time at that rate):
//                          forward        backward, x only   and the column sums   second, all three
//   65536 x 512 bf16       22-25 (26.7)   35 (40)            41                    84 (67)
//   16384 x 512 bf16       7.7 (6.7)      11 (10)            17                    23 (17)
//   131072 x 128 bf16      12.6 (13.4)    18 (20)            24                    34 (33)
//   4099 x 1001 fp32       7.7 (6.5)      12 (10)            21                    23 (16)
//   8192 x 2048 bf16       14 (13.4)      20 (20)            37                    44 (33)
//   2000 x 8000 fp32       32 (25)        39 (38)            62                    84 (64)
//   64 x 32768 bf16        9.6 (1.7)      14.6 (2.5)         14.6                  20 (4.2)
// The column sums of wide rows are what is left: few workgroups (their partial rows cost bytes) that each wait for row after row;
// asking for the next row ahead, or for two at a time, gained nothing (the wait also covers the stores in between).
#include "common.h"

namespace {

constexpr int TPB = 256;

template <typename T, int V>
struct Vec {
    T e[V];
};

// 16 bytes at the element type's own alignment (rows of odd width start anywhere; the hardware takes it)
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> ldv(const T* p) {
    Vec<T, V> v;
    __builtin_memcpy(&v, p, sizeof(v));
    return v;
}
template <typename T, int V>
__device__ __forceinline__ void stv(T* p, const Vec<T, V>& v) {
    __builtin_memcpy(p, &v, sizeof(v));
}

// A row's (or piece's) elements lane + k * TPR (in vectors) of n elements; past the end: zeros.
template <typename T, int V, int K, int TPR>
struct RowRegs {
    Vec<T, V> v[K];
    __device__ __forceinline__ void load(const T* __restrict__ p, int lane, int n) {
        const int nv = n / V, tail = n - nv * V;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int i = lane + k * TPR;
            if (nv > 0) {  // always issued, cleared afterwards: a load under a lane's condition is waited for on its own
                v[k] = ldv<T, V>(p + (int64_t)(i < nv ? i : 0) * V);
            }
            if (i >= nv) {
#pragma unroll
                for (int e = 0; e < V; ++e) v[k].e[e] = (T)0.f;
                if (i == nv) {
#pragma unroll
                    for (int e = 0; e < V - 1; ++e)
                        if (e < tail) v[k].e[e] = p[(int64_t)i * V + e];
                }
            }
        }
    }
    __device__ __forceinline__ void store(T* __restrict__ p, int lane, int n) const {
        const int nv = n / V, tail = n - nv * V;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int i = lane + k * TPR;
            if (i < nv) {
                stv<T, V>(p + (int64_t)i * V, v[k]);
            } else if (i == nv) {
#pragma unroll
                for (int e = 0; e < V - 1; ++e)
                    if (e < tail) p[(int64_t)i * V + e] = v[k].e[e];
            }
        }
    }
    __device__ __forceinline__ float at(int k, int e) const { return (float)v[k].e[e]; }
    // Between a row's sums and its results: what was computed from the elements is computed again, the packed words alone stay
    // (kept as floats beside them, a row of three bf16 tensors takes four times the registers).
    __device__ __forceinline__ void settle() {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            uint4 w = __builtin_bit_cast(uint4, v[k]);
            asm volatile("" : "+v"(w.x), "+v"(w.y), "+v"(w.z), "+v"(w.w));
            v[k] = __builtin_bit_cast(Vec<T, V>, w);
        }
    }
    // elements of vector k that exist
    static __device__ __forceinline__ int count(int k, int lane, int n) {
        const int left = n - (lane + k * TPR) * V;
        return left < 0 ? 0 : (left < V ? left : V);
    }
};

// Per-column fp32 side vectors of the same lanes; absent (NULL): `def` on the existing columns, zero behind them.
template <int V, int K, int TPR>
__device__ __forceinline__ void load_cols(const float* __restrict__ p, float def, float (&o)[K][V], int lane, int n) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int i = lane + k * TPR;
        const int left = n - i * V;
        if (p && left >= V) {
            const Vec<float, V> t = ldv<float, V>(p + (int64_t)i * V);
#pragma unroll
            for (int e = 0; e < V; ++e) o[k][e] = t.e[e];
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) o[k][e] = e < left ? (p ? p[(int64_t)i * V + e] : def) : 0.f;
        }
    }
}

// Sums over the TPR threads of a row, every thread gets them.  TPR > 64: over the whole workgroup through `lds`
// (2 * N * 16 floats; `flip` alternates its halves, so that one barrier a call is enough).
template <int N, int TPR>
__device__ __forceinline__ void row_sum(float (&s)[N], float* lds, int& flip) {
    constexpr int W = TPR < 64 ? TPR : 64;
#pragma unroll
    for (int off = W / 2; off > 0; off >>= 1) {
#pragma unroll
        for (int j = 0; j < N; ++j) s[j] += __shfl_xor(s[j], off);
    }
    if constexpr (TPR > 64) {
        constexpr int NW = TPR / 64;
        float* b = lds + flip * (N * 16);
        flip ^= 1;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int j = 0; j < N; ++j) b[j * 16 + (threadIdx.x >> 6)] = s[j];
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < N; ++j) {
            float a = 0.f;
#pragma unroll
            for (int w = 0; w < NW; ++w) a += b[j * 16 + w];
            s[j] = a;
        }
    }
}

// Side vectors of a kernel whose threads walk over many rows stay in registers (HOLD); where a row takes 512 threads and more,
// registers are short and they are read again for each row, vector by vector.
template <int V, int K, int TPR, bool HOLD>
struct Cols {
    float held[HOLD ? K : 1][V];
    const float* p;
    float def;
    __device__ __forceinline__ Cols(const float* p_, float def_, int lane, int n) : p(p_), def(def_) {
        if constexpr (HOLD) load_cols<V, K, TPR>(p_, def_, held, lane, n);
    }
    __device__ __forceinline__ void get(int k, int lane, int n, float (&o)[V]) const {
        if constexpr (HOLD) {
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = held[k][e];
        } else {
            float one[1][V];
            load_cols<V, 1, TPR>(p ? p + (int64_t)k * TPR * V : nullptr, def, one, lane, n - k * TPR * V);
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = one[0][e];
        }
    }
};

struct RowArgs {
    const void *x, *g, *v;
    const float *w, *b, *cw, *cb;
    void *y, *y2;      // forward: y.  backward: gx.  second: gg, gxx
    float2* stats;     // (m, r) of each row (forward: may be NULL)
    float2* vstats;    // second: (mean v, mean(v t)) of each row, for the column kernel (may be NULL)
    float* part;       // column partials [blocks][ncol][D], or NULL
    float* join;       // long rows: partial sums [rows][pieces][NSUM]
    int64_t rows;
    int D;
    float eps;
    int pieces, piece;  // long rows: pieces per row, elements in each but the last
    int row_blocks, col_tiles;  // backward in one launch with its column sums: workgroups of the rows, tiles of columns
    int64_t chunk;              // and rows in a chunk
};

template <int TPR>
constexpr int block_of() {
    return TPR <= TPB ? TPB : TPR;
}

// ---- forward -----------------------------------------------------------------------------------------------------
template <typename T, int TPR, int K>
__global__ void __launch_bounds__(block_of<TPR>()) ln_fwd_k(const RowArgs a) {
    constexpr int V = VecOf<T>::V, BLK = block_of<TPR>(), G = BLK / TPR;
    __shared__ float lds[2 * 16];
    int flip = 0;
    const int lane = threadIdx.x % TPR, grp = threadIdx.x / TPR;
    const int D = a.D;
    const Cols<V, K, TPR, (TPR < 512)> w(a.w, 1.f, lane, D), b(a.b, 0.f, lane, D);
    const float inv = 1.f / (float)D;
    for (int64_t row = (int64_t)blockIdx.x * G + grp; row < a.rows; row += (int64_t)gridDim.x * G) {
        RowRegs<T, V, K, TPR> x;
        x.load((const T*)a.x + row * D, lane, D);
        float s[1] = {0.f};
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) s[0] += x.at(k, e);
        row_sum<1, TPR>(s, lds, flip);
        x.settle();
        const float m = s[0] / (float)D;  // (a division: a row of one value has that mean, and 1 / r may be 300 times the rounding)
        float q[1] = {0.f};
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int cnt = RowRegs<T, V, K, TPR>::count(k, lane, D);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float d = e < cnt ? x.at(k, e) - m : 0.f;
                q[0] = fmaf(d, d, q[0]);
            }
        }
        row_sum<1, TPR>(q, lds, flip);
        x.settle();
        const float r = rsqrtf(q[0] * inv + a.eps);
        if (a.stats && lane == 0) a.stats[row] = make_float2(m, r);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float wk[V], bk[V];
            w.get(k, lane, D, wk);
            b.get(k, lane, D, bk);
#pragma unroll
            for (int e = 0; e < V; ++e) x.v[k].e[e] = (T)fmaf((x.at(k, e) - m) * r, wk[e], bk[e]);
        }
        x.store((T*)a.y + row * D, lane, D);
    }
}

// Column sums of the row groups of one workgroup: of a wave's groups by exchange between lanes, of the waves through LDS in their
// order, then written as the workgroup's partial row.  (One group after another through LDS: 12 us of the 38 that the pass over
// 131072 x 128 bf16 takes; like this 2.)
template <int NC, int V, int K, int TPR>
__device__ __forceinline__ void write_partials(float (&acc)[NC][K][V], float* part, int lane, int D) {
    constexpr int G = block_of<TPR>() / TPR, W = TPB / 64, DP = K * TPR * V;
    float* out = part + (int64_t)blockIdx.x * NC * D;
    if constexpr (G == 1) {
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const int c = (lane + k * TPR) * V + e;
                    if (c < D) out[(int64_t)j * D + c] = acc[j][k][e];
                }
    } else {
        __shared__ __attribute__((aligned(16))) float cols[W][NC][DP];
        const int wave = threadIdx.x >> 6;
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int k = 0; k < K; ++k) {
#pragma unroll
                for (int e = 0; e < V; ++e)
#pragma unroll
                    for (int off = TPR; off < 64; off *= 2) acc[j][k][e] += __shfl_xor(acc[j][k][e], off);
                if ((threadIdx.x & 63) < TPR) {
#pragma unroll
                    for (int e = 0; e < V; ++e) cols[wave][j][(lane + k * TPR) * V + e] = acc[j][k][e];
                }
            }
        __syncthreads();
        for (int i = threadIdx.x; i < NC * DP; i += TPB) {
            const int j = i / DP, c = i % DP;
            float s = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) s += cols[w][j][c];
            if (c < D) out[(int64_t)j * D + c] = s;
        }
    }
}

// ---- column sums down the rows -------------------------------------------------------------------------------------
// 16 lanes across a vector of columns each, the workgroup's other threads down the rows of chunk `chunk_id`.  PASS 1: (g t, g),
// 2: g r P(v).  out: [chunks][NC][D].
template <typename T, int PASS, int BLK>
__device__ __forceinline__ void col_sums(const RowArgs& a, float* __restrict__ out, int64_t chunk, int tile, int chunk_id) {
    constexpr int V = VecOf<T>::V, NC = PASS == 1 ? 2 : 1, CG = BLK / 16, NW = BLK / 64;
    __shared__ float red[NC][NW][16 * V];
    const int lane = threadIdx.x & 15, grp = threadIdx.x >> 4, wave = threadIdx.x >> 6;
    const int c0 = (tile * 16 + lane) * V;
    const int left = a.D - c0;
    float acc[NC][V];
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) acc[j][e] = 0.f;
    const int64_t r0 = (int64_t)chunk_id * chunk, r1 = r0 + chunk < a.rows ? r0 + chunk : a.rows;
    for (int64_t row = r0 + grp; row < r1; row += CG) {
        const float2 st = a.stats[row];
        const float2 vs = PASS == 2 ? a.vstats[row] : make_float2(0.f, 0.f);
        Vec<T, V> x, g, v;
        const int64_t at = row * a.D + c0;
        if (left >= V) {
            x = ldv<T, V>((const T*)a.x + at);
            g = ldv<T, V>((const T*)a.g + at);
            if (PASS == 2) v = ldv<T, V>((const T*)a.v + at);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                x.e[e] = e < left ? ((const T*)a.x)[at + e] : (T)0.f;
                g.e[e] = e < left ? ((const T*)a.g)[at + e] : (T)0.f;
                if (PASS == 2) v.e[e] = e < left ? ((const T*)a.v)[at + e] : (T)0.f;
            }
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float t = ((float)x.e[e] - st.x) * st.y, gv = (float)g.e[e];
            if constexpr (PASS == 1) {
                acc[0][e] = fmaf(gv, t, acc[0][e]);
                acc[1][e] += gv;
            } else {
                acc[0][e] = fmaf(gv, st.y * ((float)v.e[e] - vs.x - t * vs.y), acc[0][e]);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) {
            acc[j][e] += __shfl_xor(acc[j][e], 16);
            acc[j][e] += __shfl_xor(acc[j][e], 32);
            if ((threadIdx.x & 63) < 16) red[j][wave][lane * V + e] = acc[j][e];
        }
    __syncthreads();
    for (int i = threadIdx.x; i < NC * 16 * V; i += BLK) {
        const int j = i / (16 * V), c = i % (16 * V), col = tile * 16 * V + c;
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < NW; ++k) s += red[j][k][c];
        if (col < a.D) out[((int64_t)chunk_id * NC + j) * a.D + col] = s;
    }
}

template <typename T, int PASS>
__global__ void __launch_bounds__(TPB) ln_cols_k(const RowArgs a, float* __restrict__ out, int64_t chunk, int tiles) {
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {  // (once, up to COL_TILES of them)
        if (tile != (int)blockIdx.x) __syncthreads();
        col_sums<T, PASS, TPB>(a, out, chunk, tile, blockIdx.y);
    }
}

// ---- backward ----------------------------------------------------------------------------------------------------
// COLS 1: column sums kept by the threads.  2: the workgroups behind `a.row_blocks` sum the columns down the rows (they need the
// forward's statistics only), in the same launch.
template <typename T, int TPR, int K, int COLS>
__global__ void __launch_bounds__(block_of<TPR>()) ln_bwd_k(const RowArgs a) {
    constexpr int V = VecOf<T>::V, BLK = block_of<TPR>(), G = BLK / TPR;
    if constexpr (COLS == 2) {
        if ((int)blockIdx.x >= a.row_blocks) {
            const int i = (int)blockIdx.x - a.row_blocks;
            col_sums<T, 1, BLK>(a, a.part, a.chunk, i % a.col_tiles, i / a.col_tiles);
            return;
        }
    }
    __shared__ float lds[2 * 2 * 16];
    int flip = 0;
    const int lane = threadIdx.x % TPR, grp = threadIdx.x / TPR;
    const int D = a.D, blocks = COLS == 2 ? a.row_blocks : (int)gridDim.x;
    const Cols<V, K, TPR, (TPR < 512)> w(a.w, 1.f, lane, D);
    float acc[2][COLS == 1 ? K : 1][V];
    if (COLS == 1) {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) acc[0][k][e] = acc[1][k][e] = 0.f;
    }
    const float inv = 1.f / (float)D;
    for (int64_t row = (int64_t)blockIdx.x * G + grp; row < a.rows; row += (int64_t)blocks * G) {
        RowRegs<T, V, K, TPR> x, g;
        x.load((const T*)a.x + row * D, lane, D);
        g.load((const T*)a.g + row * D, lane, D);
        const float2 st = a.stats[row];
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float wk[V];
            w.get(k, lane, D, wk);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float gv = g.at(k, e), t = (x.at(k, e) - st.x) * st.y, h = gv * wk[e];
                s[0] += h;
                s[1] = fmaf(h, t, s[1]);
                if (COLS == 1) {
                    acc[0][k][e] = fmaf(gv, t, acc[0][k][e]);
                    acc[1][k][e] += gv;
                }
            }
        }
        if (a.y) {
            row_sum<2, TPR>(s, lds, flip);
            x.settle();
            g.settle();
            const float s1 = s[0] * inv, s2 = s[1] * inv;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                float wk[V];
                w.get(k, lane, D, wk);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float t = (x.at(k, e) - st.x) * st.y;
                    g.v[k].e[e] = (T)(st.y * (g.at(k, e) * wk[e] - s1 - t * s2));
                }
            }
            g.store((T*)a.y + row * D, lane, D);
        }
    }
    if constexpr (COLS == 1) write_partials<2, V, K, TPR>(acc, a.part, lane, D);
}

// ---- second order ------------------------------------------------------------------------------------------------
// The row sums of the second pass: v, v t, h, h t, v h, q, q t with q = g cw.
constexpr int NS2 = 7;

__device__ __forceinline__ void second_sums(float x, float g, float v, float w, float cw, float2 st, float (&s)[NS2]) {
    const float t = (x - st.x) * st.y, h = g * w, q = g * cw;
    s[0] += v;
    s[1] = fmaf(v, t, s[1]);
    s[2] += h;
    s[3] = fmaf(h, t, s[3]);
    s[4] = fmaf(v, h, s[4]);
    s[5] += q;
    s[6] = fmaf(q, t, s[6]);
}

struct SecondRow {
    float m, r, vm, vt, ht, um, ut, rs;
    __device__ __forceinline__ SecondRow(float2 st, const float (&s)[NS2], float inv) {
        m = st.x;
        r = st.y;
        vm = s[0] * inv;
        vt = s[1] * inv;
        const float hm = s[2] * inv;
        ht = s[3] * inv;
        um = fmaf(-r, vm * ht + hm * vt, s[5] * inv);
        ut = fmaf(-2.f * r, ht * vt, s[6] * inv);
        rs = r * (s[4] * inv - vm * hm - vt * ht);
    }
    // gxx, gg and g r P(v) of one element
    __device__ __forceinline__ void at(float x, float g, float v, float w, float cw, float cb, float& gxx, float& gg, float& gw) const {
        const float t = (x - m) * r, pv = r * (v - vm - t * vt);
        const float u = fmaf(-r, v * ht + g * w * vt, g * cw);
        gxx = r * (u - um - t * (ut + rs));
        gg = fmaf(w, pv, fmaf(cw, t, cb));
        gw = g * pv;
    }
};

template <typename T, int TPR, int K, int COLS, bool CC>  // CC: cotangents of the column sums are there
__global__ void __launch_bounds__(block_of<TPR>()) ln_bwd2_k(const RowArgs a) {
    constexpr int V = VecOf<T>::V, BLK = block_of<TPR>(), G = BLK / TPR;
    __shared__ float lds[2 * NS2 * 16];
    int flip = 0;
    const int lane = threadIdx.x % TPR, grp = threadIdx.x / TPR;
    const int D = a.D;
    float acc[1][COLS == 1 ? K : 1][V];
    if (COLS == 1) {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) acc[0][k][e] = 0.f;
    }
    const Cols<V, K, TPR, false> w(a.w, 1.f, lane, D), cw(a.cw, 0.f, lane, D), cb(a.cb, 0.f, lane, D);
    const float inv = 1.f / (float)D;
    for (int64_t row = (int64_t)blockIdx.x * G + grp; row < a.rows; row += (int64_t)gridDim.x * G) {
        RowRegs<T, V, K, TPR> x, g, v;
        x.load((const T*)a.x + row * D, lane, D);
        g.load((const T*)a.g + row * D, lane, D);
        v.load((const T*)a.v + row * D, lane, D);
        const float2 st = a.stats[row];
        float s[NS2] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float wk[V], cwk[V];
            w.get(k, lane, D, wk);
            if (CC) cw.get(k, lane, D, cwk);
#pragma unroll
            for (int e = 0; e < V; ++e) second_sums(x.at(k, e), g.at(k, e), v.at(k, e), wk[e], CC ? cwk[e] : 0.f, st, s);
        }
        row_sum<NS2, TPR>(s, lds, flip);
        x.settle();
        g.settle();
        v.settle();
        const SecondRow sr(st, s, inv);
        if (a.vstats && lane == 0) a.vstats[row] = make_float2(sr.vm, sr.vt);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float wk[V], cwk[V], cbk[V];
            w.get(k, lane, D, wk);
            if (CC) {
                cw.get(k, lane, D, cwk);
                cb.get(k, lane, D, cbk);
            }
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float gxx, gg, gw;
                sr.at(x.at(k, e), g.at(k, e), v.at(k, e), wk[e], CC ? cwk[e] : 0.f, CC ? cbk[e] : 0.f, gxx, gg, gw);
                x.v[k].e[e] = (T)gxx;
                v.v[k].e[e] = (T)gg;
                if (COLS == 1) acc[0][k][e] += gw;
            }
        }
        if (a.y) v.store((T*)a.y + row * D, lane, D);
        if (a.y2) x.store((T*)a.y2 + row * D, lane, D);
    }
    if constexpr (COLS == 1) write_partials<1, V, K, TPR>(acc, a.part, lane, D);
}

// ---- long rows: pieces of a row sum, then join and write -----------------------------------------------------------
// PASS 0: forward (join: (mean, centred second moment) of each piece), 1: backward (2 sums), 2: second (7 sums)
constexpr int LK = 4;
template <int PASS>
constexpr int join_n() {
    return PASS == 2 ? NS2 : 2;
}

template <typename T, int PASS>
__global__ void __launch_bounds__(TPB) ln_long_sum_k(const RowArgs a) {
    constexpr int V = VecOf<T>::V, N = join_n<PASS>();
    __shared__ float lds[2 * N * 16];
    int flip = 0;
    const int64_t row = blockIdx.x / a.pieces;
    const int p = blockIdx.x % a.pieces, lane = threadIdx.x;
    const int64_t at = row * a.D + (int64_t)p * a.piece;
    const int n = min(a.piece, a.D - p * a.piece);
    float* out = a.join + (row * a.pieces + p) * N;
    RowRegs<T, V, LK, TPB> x, g, v;
    x.load((const T*)a.x + at, lane, n);
    if constexpr (PASS == 0) {
        float s[1] = {0.f}, q[1] = {0.f};
#pragma unroll
        for (int k = 0; k < LK; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) s[0] += x.at(k, e);
        row_sum<1, TPB>(s, lds, flip);
        const float m = s[0] / (float)n;
#pragma unroll
        for (int k = 0; k < LK; ++k) {
            const int cnt = RowRegs<T, V, LK, TPB>::count(k, lane, n);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float d = e < cnt ? x.at(k, e) - m : 0.f;
                q[0] = fmaf(d, d, q[0]);
            }
        }
        row_sum<1, TPB>(q, lds, flip);
        if (lane == 0) {
            out[0] = m;
            out[1] = q[0];
        }
    } else {
        g.load((const T*)a.g + at, lane, n);
        const float2 st = a.stats[row];
        float w[LK][V], s[N];
        load_cols<V, LK, TPB>(a.w ? a.w + (int64_t)p * a.piece : nullptr, 1.f, w, lane, n);
#pragma unroll
        for (int j = 0; j < N; ++j) s[j] = 0.f;
        if constexpr (PASS == 1) {
#pragma unroll
            for (int k = 0; k < LK; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float t = (x.at(k, e) - st.x) * st.y, h = g.at(k, e) * w[k][e];
                    s[0] += h;
                    s[1] = fmaf(h, t, s[1]);
                }
        } else {
            float cw[LK][V];
            v.load((const T*)a.v + at, lane, n);
            load_cols<V, LK, TPB>(a.cw ? a.cw + (int64_t)p * a.piece : nullptr, 0.f, cw, lane, n);
#pragma unroll
            for (int k = 0; k < LK; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) second_sums(x.at(k, e), g.at(k, e), v.at(k, e), w[k][e], cw[k][e], st, s);
        }
        row_sum<N, TPB>(s, lds, flip);
        if (lane == 0) {
#pragma unroll
            for (int j = 0; j < N; ++j) out[j] = s[j];
        }
    }
}

template <typename T, int PASS>
__global__ void __launch_bounds__(TPB) ln_long_apply_k(const RowArgs a) {
    constexpr int V = VecOf<T>::V, N = join_n<PASS>();
    __shared__ float lds[2 * N * 16];
    int flip = 0;
    const int64_t row = blockIdx.x / a.pieces;
    const int p = blockIdx.x % a.pieces, lane = threadIdx.x;
    const int64_t at = row * a.D + (int64_t)p * a.piece;
    const int n = min(a.piece, a.D - p * a.piece);
    const float* in = a.join + row * a.pieces * N;
    const float inv = 1.f / (float)a.D;
    RowRegs<T, V, LK, TPB> x, g, v;
    x.load((const T*)a.x + at, lane, n);
    float w[LK][V];
    load_cols<V, LK, TPB>(a.w ? a.w + (int64_t)p * a.piece : nullptr, 1.f, w, lane, n);
    if constexpr (PASS == 0) {
        float s[1] = {0.f}, q[1] = {0.f};
        for (int i = lane; i < a.pieces; i += TPB) s[0] = fmaf((float)min(a.piece, a.D - i * a.piece), in[i * N], s[0]);
        row_sum<1, TPB>(s, lds, flip);
        const float m = s[0] / (float)a.D;
        for (int i = lane; i < a.pieces; i += TPB) {  // second moments about the pieces' means, moved to the row's
            const float d = in[i * N] - m;
            q[0] += fmaf((float)min(a.piece, a.D - i * a.piece) * d, d, in[i * N + 1]);
        }
        row_sum<1, TPB>(q, lds, flip);
        const float r = rsqrtf(q[0] * inv + a.eps);
        if (a.stats && p == 0 && lane == 0) a.stats[row] = make_float2(m, r);
        float b[LK][V];
        load_cols<V, LK, TPB>(a.b ? a.b + (int64_t)p * a.piece : nullptr, 0.f, b, lane, n);
#pragma unroll
        for (int k = 0; k < LK; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) x.v[k].e[e] = (T)fmaf((x.at(k, e) - m) * r, w[k][e], b[k][e]);
        x.store((T*)a.y + at, lane, n);
    } else {
        g.load((const T*)a.g + at, lane, n);
        const float2 st = a.stats[row];
        float s[N];
#pragma unroll
        for (int j = 0; j < N; ++j) s[j] = 0.f;
        for (int i = lane; i < a.pieces; i += TPB) {
#pragma unroll
            for (int j = 0; j < N; ++j) s[j] += in[i * N + j];
        }
        row_sum<N, TPB>(s, lds, flip);
        if constexpr (PASS == 1) {
            const float s1 = s[0] * inv, s2 = s[1] * inv;
#pragma unroll
            for (int k = 0; k < LK; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float t = (x.at(k, e) - st.x) * st.y;
                    g.v[k].e[e] = (T)(st.y * (g.at(k, e) * w[k][e] - s1 - t * s2));
                }
            g.store((T*)a.y + at, lane, n);
        } else {
            const SecondRow sr(st, s, inv);
            if (a.vstats && p == 0 && lane == 0) a.vstats[row] = make_float2(sr.vm, sr.vt);
            v.load((const T*)a.v + at, lane, n);
            float cw[LK][V], cb[LK][V];
            load_cols<V, LK, TPB>(a.cw ? a.cw + (int64_t)p * a.piece : nullptr, 0.f, cw, lane, n);
            load_cols<V, LK, TPB>(a.cb ? a.cb + (int64_t)p * a.piece : nullptr, 0.f, cb, lane, n);
#pragma unroll
            for (int k = 0; k < LK; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    float gxx, gg, gw;
                    sr.at(x.at(k, e), g.at(k, e), v.at(k, e), w[k][e], cw[k][e], cb[k][e], gxx, gg, gw);
                    x.v[k].e[e] = (T)gxx;
                    v.v[k].e[e] = (T)gg;
                }
            if (a.y) v.store((T*)a.y + at, lane, n);
            if (a.y2) x.store((T*)a.y2 + at, lane, n);
        }
    }
}

// out[c] = sum_p part[p][c] over `n` partial rows of `width` columns, in a fixed order: 16 columns x 64 slices a workgroup.
// The first `split` columns go to out0, the others to out1 (either may be NULL).
__global__ void __launch_bounds__(1024) fold_cols_k(const float* __restrict__ part, int n, int64_t width, float* __restrict__ out0,
                                                    float* __restrict__ out1, int64_t split) {
    __shared__ float red[16][17];
    constexpr int AHEAD = 8;  // rows requested at a time
    const int c = threadIdx.x & 15, sl = threadIdx.x >> 4;
    const int64_t col = (int64_t)blockIdx.x * 16 + c, in = col < width ? col : 0;
    float s = 0.f;
    for (int p = sl; p < n; p += 64 * AHEAD) {
        float v[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) v[k] = part[(int64_t)(p + 64 * k < n ? p + 64 * k : p) * width + in];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) s += p + 64 * k < n ? v[k] : 0.f;
    }
    s += __shfl_xor(s, 16);
    s += __shfl_xor(s, 32);
    if ((threadIdx.x & 63) < 16) red[threadIdx.x >> 6][c] = s;
    __syncthreads();
    if (sl == 0 && col < width) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < 16; ++k) t += red[k][c];
        if (col < split) {
            if (out0) out0[col] = t;
        } else if (out1) {
            out1[col - split] = t;
        }
    }
}

// ---- launch plan ---------------------------------------------------------------------------------------------------
struct Plan {
    int tpr, k;      // threads per row, vectors per thread; tpr = 0: long rows
    int blocks;      // row kernels
    bool fused;      // column sums kept by the row kernel
    int chunks;      // column kernel: chunks of rows
    int64_t chunk;
    int pieces, piece;
    int64_t floats;  // workspace
};

// Four workgroups of 256 threads a CU; forward, with fewer registers, eight (65536 x 512 bf16: 23.8 us against 26.5).
constexpr int MAXB = 1024;
// Tiles of columns side by side in a launch (work items are counted in 32 bits: 2^24 workgroups of 256, fp32 rows of 2^30, are one too many)
constexpr int COL_TILES = 1 << 23;

// pass 0 forward, 1 backward, 2 second.  cols: column sums wanted.
Plan plan_of(int64_t rows, int64_t D, int dtype, int pass, bool cols) {
    Plan p = {};
    const int V = dtype == GAN_F32 ? 4 : 8;
    const int64_t nv = (D + V - 1) / V;
    const int ncol = pass == 2 ? 1 : 2;
    if (nv <= 64) {
        p.tpr = nv <= 16 ? 16 : 64;
        p.k = 1;
    } else if (nv <= 512) {
        p.tpr = nv <= 128 ? 64 : 256;
        p.k = nv <= 128 || nv > 256 ? 2 : 1;
    } else if (nv <= (pass == 2 ? 2048 : 4096)) {  // (three tensors of a row in 1024 threads' 128 registers spill)
        p.tpr = nv <= 1024 || pass == 2 ? 512 : 1024;
        p.k = nv <= 1024 || (nv <= 2048 && pass < 2) ? 2 : 4;
    }
    if (p.tpr) {
        const int g = p.tpr >= TPB ? 1 : TPB / p.tpr;
        const int64_t need = ceil_div64(rows, g);
        const int64_t many = pass == 0 ? 2 * MAXB : MAXB;
        p.blocks = (int)(need < many ? need : many);
        if (cols && pass > 0 && p.tpr <= 512) {
            // A partial row of ncol D floats per workgroup is written and read again, next to at least three tensor rows of D
            // elements that a row costs anyway: few enough workgroups keep that under a sixth (second order, with one partial row
            // against five tensors: twice as many, 8192 x 2048 bf16 54 -> 45 us; rows of 512 threads lose by it, 84 -> 90).  Where so
            // few are left that they would not fill the chip, a kernel down the columns reads the tensors a second time instead.
            const int64_t most = rows / ((dtype == GAN_F32 ? 8 : 16) / (pass == 2 && p.tpr <= 256 ? 2 : 1));
            if (most >= 64) {
                p.fused = true;
                if (p.blocks > most) p.blocks = (int)most;
                p.floats = (int64_t)p.blocks * ncol * D;
            }
        }
    } else {
        p.piece = TPB * LK * V;
        p.pieces = (int)ceil_div64(D, p.piece);
        p.floats = rows * p.pieces * (pass == 2 ? NS2 : 2);
    }
    if (cols && pass > 0 && !p.fused) {
        const int64_t tiles = ceil_div64(D, 16 * V);
        int64_t chunks = ceil_div64(512, tiles);  // two workgroups a CU, at least 64 rows in each
        const int64_t most = ceil_div64(rows, 64);
        if (chunks > most) chunks = most;
        if (chunks < 1) chunks = 1;
        p.chunk = ceil_div64(rows, chunks);
        p.chunks = (int)ceil_div64(rows, p.chunk);
        if (p.chunks > 1) p.floats += (int64_t)p.chunks * ncol * D;
        if (pass == 2) p.floats += 2 * rows + 2;  // vstats
    }
    return p;
}

// (work items of a launch are counted in 32 bits, 256 in a workgroup)
bool too_many(int64_t rows, const Plan& p) { return !p.tpr && rows * p.pieces >= (1LL << 24); }

template <typename T, int PASS, int COLS, int TPR, int K>
void launch_row(int blocks, const RowArgs& a, hipStream_t st) {
    constexpr int BLK = block_of<TPR>();
    if constexpr (PASS == 0)
        hipLaunchKernelGGL((ln_fwd_k<T, TPR, K>), dim3(blocks), dim3(BLK), 0, st, a);
    else if constexpr (PASS == 1)
        hipLaunchKernelGGL((ln_bwd_k<T, TPR, K, COLS>), dim3(blocks), dim3(BLK), 0, st, a);
    else if (a.cw || a.cb)
        hipLaunchKernelGGL((ln_bwd2_k<T, TPR, K, COLS, true>), dim3(blocks), dim3(BLK), 0, st, a);
    else
        hipLaunchKernelGGL((ln_bwd2_k<T, TPR, K, COLS, false>), dim3(blocks), dim3(BLK), 0, st, a);
}

template <typename T, int PASS, int COLS>
void launch_rows(const Plan& p, int blocks, const RowArgs& a, hipStream_t st) {
    switch (p.tpr * 8 + p.k) {
        case 16 * 8 + 1: return launch_row<T, PASS, COLS, 16, 1>(blocks, a, st);
        case 64 * 8 + 1: return launch_row<T, PASS, COLS, 64, 1>(blocks, a, st);
        case 64 * 8 + 2: return launch_row<T, PASS, COLS, 64, 2>(blocks, a, st);
        case 256 * 8 + 1: return launch_row<T, PASS, COLS, 256, 1>(blocks, a, st);
        case 256 * 8 + 2: return launch_row<T, PASS, COLS, 256, 2>(blocks, a, st);
        case 512 * 8 + 2: return launch_row<T, PASS, COLS, 512, 2>(blocks, a, st);
    }
    if constexpr (PASS == 2) {
        launch_row<T, PASS, COLS, 512, 4>(blocks, a, st);
    } else if constexpr (COLS != 1) {
        if (p.k == 2) launch_row<T, PASS, COLS, 1024, 2>(blocks, a, st);
        else launch_row<T, PASS, COLS, 1024, 4>(blocks, a, st);
    }
}

template <typename T, int PASS>
int run_pass(const Plan& p, RowArgs a, float* gw, float* gb, float* ws, hipStream_t st) {
    constexpr int NC = PASS == 2 ? 1 : 2;
    const int64_t D = a.D;
    const bool cols = PASS > 0 && (gw || gb);
    float* at = ws;
    const bool rows_out = PASS == 0 || a.y || a.y2 || (PASS == 2 && cols);
    if (p.tpr) {
        if (p.fused) {
            a.part = at;
            at += (int64_t)p.blocks * NC * D;
            if constexpr (PASS > 0) launch_rows<T, PASS, 1>(p, p.blocks, a, st);
            GAN_CHECK_LAUNCH("layernorm");
            hipLaunchKernelGGL(fold_cols_k, dim3((unsigned)ceil_div64(NC * D, 16)), dim3(1024), 0, st, a.part, p.blocks, (int64_t)NC * D, gw, gb, D);
            GAN_CHECK_LAUNCH("layernorm(fold)");
            return GAN_OK;
        }
    } else {
        a.join = at;
        a.pieces = p.pieces;
        a.piece = p.piece;
        at += a.rows * p.pieces * join_n<PASS>();
    }
    if (PASS == 2 && cols) {
        at += (2 - (at - ws) % 2) % 2;
        a.vstats = (float2*)at;
        at += 2 * a.rows;
    }
    bool summed = !cols;
    float* const sums = p.chunks > 1 ? at : gw;  // one chunk: the kernel's [NC][D] are the gradients
    if (rows_out) {
        if (p.tpr) {
            if constexpr (PASS == 1) {
                if (cols) {  // the columns in the same launch: tiles of them behind the rows' workgroups
                    a.row_blocks = p.blocks;
                    a.col_tiles = (int)ceil_div64(D, 16 * VecOf<T>::V);
                    a.chunk = p.chunk;
                    a.part = sums;
                    launch_rows<T, 1, 2>(p, p.blocks + a.col_tiles * p.chunks, a, st);
                    summed = true;
                } else {
                    launch_rows<T, 1, 0>(p, p.blocks, a, st);
                }
            } else {
                launch_rows<T, PASS, 0>(p, p.blocks, a, st);
            }
        } else {
            const dim3 grid((unsigned)(a.rows * p.pieces));
            hipLaunchKernelGGL((ln_long_sum_k<T, PASS>), grid, dim3(TPB), 0, st, a);
            GAN_CHECK_LAUNCH("layernorm(sum)");
            hipLaunchKernelGGL((ln_long_apply_k<T, PASS>), grid, dim3(TPB), 0, st, a);
        }
        GAN_CHECK_LAUNCH("layernorm(rows)");
    }
    if constexpr (PASS > 0) {
        if (!summed) {
            const int tiles = (int)ceil_div64(D, 16 * VecOf<T>::V);
            const dim3 grid((unsigned)(tiles < COL_TILES ? tiles : COL_TILES), (unsigned)p.chunks);
            hipLaunchKernelGGL((ln_cols_k<T, PASS>), grid, dim3(TPB), 0, st, a, sums, p.chunk, tiles);
            GAN_CHECK_LAUNCH("layernorm(columns)");
        }
        if (cols && p.chunks > 1) {
            hipLaunchKernelGGL(fold_cols_k, dim3((unsigned)ceil_div64(NC * D, 16)), dim3(1024), 0, st, sums, p.chunks, (int64_t)NC * D, gw, gb, D);
            GAN_CHECK_LAUNCH("layernorm(fold)");
        }
    }
    return GAN_OK;
}

int check_common(const char* what, int64_t rows, int64_t D, int dtype, float* ws, int64_t ws_floats, const Plan& p) {
    GAN_CHECK_ARG(!too_many(rows, p), "%s: too many rows", what);
    GAN_CHECK_ARG(p.floats == 0 || (ws && ws_floats >= p.floats), "%s: workspace of %lld floats wanted, %lld given", what, (long long)p.floats,
                  (long long)(ws ? ws_floats : 0));
    GAN_CHECK_ARG(((uintptr_t)ws % 16) == 0, "%s: workspace must be 16-byte aligned", what);
    return GAN_OK;
}

bool bad_shape(int64_t rows, int64_t D, int dtype) {
    return rows < 0 || rows >= (1LL << 31) || D <= 0 || D > (1 << 30) || (dtype != GAN_F32 && dtype != GAN_BF16);
}

}  // namespace

extern "C" int64_t gan_layernorm_workspace(int64_t rows, int64_t D, int dtype, int pass, int columns) {
    if (bad_shape(rows, D, dtype) || pass < 0 || pass > 2) return -1;
    const Plan p = plan_of(rows ? rows : 1, D, dtype, pass, columns != 0);
    return !rows ? 0 : too_many(rows, p) ? -1 : p.floats;
}

extern "C" int gan_layernorm_fwd(const void* x, const float* w, const float* b, void* y, float* stats, int64_t rows, int64_t D, float eps,
                                 int dtype, float* ws, int64_t ws_floats, gan_stream_t stream) {
    GAN_CHECK_ARG(!bad_shape(rows, D, dtype), "layernorm_fwd: bad shape or dtype (%lld rows of %lld, dtype %d)", (long long)rows, (long long)D, dtype);
    GAN_CHECK_ARG(eps >= 0.f, "layernorm_fwd: eps must not be negative");
    if (rows == 0) return GAN_OK;
    GAN_CHECK_ARG(x && y, "layernorm_fwd: null pointer");
    GAN_CHECK_ARG(((uintptr_t)stats % 8) == 0, "layernorm_fwd: stats must be 8-byte aligned");
    const Plan p = plan_of(rows, D, dtype, 0, false);
    if (int rc = check_common("layernorm_fwd", rows, D, dtype, ws, ws_floats, p)) return rc;
    RowArgs a = {};
    a.x = x; a.w = w; a.b = b; a.y = y; a.stats = (float2*)stats; a.rows = rows; a.D = (int)D; a.eps = eps;
    return dtype == GAN_F32 ? run_pass<float, 0>(p, a, nullptr, nullptr, ws, (hipStream_t)stream)
                            : run_pass<bf16, 0>(p, a, nullptr, nullptr, ws, (hipStream_t)stream);
}

extern "C" int gan_layernorm_bwd(const void* g, const void* x, const float* w, const float* stats, void* gx, float* gwb, int64_t rows, int64_t D,
                                 int dtype, float* ws, int64_t ws_floats, gan_stream_t stream) {
    GAN_CHECK_ARG(!bad_shape(rows, D, dtype), "layernorm_bwd: bad shape or dtype (%lld rows of %lld, dtype %d)", (long long)rows, (long long)D, dtype);
    GAN_CHECK_ARG(rows > 0, "layernorm_bwd: no rows");
    GAN_CHECK_ARG(g && x && stats, "layernorm_bwd: null pointer");
    GAN_CHECK_ARG(((uintptr_t)stats % 8) == 0, "layernorm_bwd: stats must be 8-byte aligned");
    const Plan p = plan_of(rows, D, dtype, 1, gwb != nullptr);
    if (int rc = check_common("layernorm_bwd", rows, D, dtype, ws, ws_floats, p)) return rc;
    RowArgs a = {};
    a.x = x; a.g = g; a.w = w; a.y = gx; a.stats = (float2*)stats; a.rows = rows; a.D = (int)D;
    float* gb = gwb ? gwb + D : nullptr;
    return dtype == GAN_F32 ? run_pass<float, 1>(p, a, gwb, gb, ws, (hipStream_t)stream) : run_pass<bf16, 1>(p, a, gwb, gb, ws, (hipStream_t)stream);
}

extern "C" int gan_layernorm_bwd2(const void* v, const float* cw, const float* cb, const void* g, const void* x, const float* w,
                                  const float* stats, void* gg, void* gxx, float* gww, int64_t rows, int64_t D, int dtype, float* ws,
                                  int64_t ws_floats, gan_stream_t stream) {
    GAN_CHECK_ARG(!bad_shape(rows, D, dtype), "layernorm_bwd2: bad shape or dtype (%lld rows of %lld, dtype %d)", (long long)rows, (long long)D, dtype);
    GAN_CHECK_ARG(rows > 0, "layernorm_bwd2: no rows");
    GAN_CHECK_ARG(v && g && x && stats, "layernorm_bwd2: null pointer");
    GAN_CHECK_ARG(((uintptr_t)stats % 8) == 0, "layernorm_bwd2: stats must be 8-byte aligned");
    const Plan p = plan_of(rows, D, dtype, 2, gww != nullptr);
    if (int rc = check_common("layernorm_bwd2", rows, D, dtype, ws, ws_floats, p)) return rc;
    RowArgs a = {};
    a.x = x; a.g = g; a.v = v; a.w = w; a.cw = cw; a.cb = cb; a.y = gg; a.y2 = gxx; a.stats = (float2*)stats; a.rows = rows; a.D = (int)D;
    return dtype == GAN_F32 ? run_pass<float, 2>(p, a, gww, nullptr, ws, (hipStream_t)stream)
                            : run_pass<bf16, 2>(p, a, gww, nullptr, ws, (hipStream_t)stream);
}
