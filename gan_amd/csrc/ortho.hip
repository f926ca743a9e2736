// Newton-Schulz orthogonalisation of matrices and the optimiser step built on it (gfx950).
//   X = G / max(|G|, eps) (Frobenius norm; X is m x n with m <= n, a tall G is worked on as its transpose), then `steps` times
//   A = X X',  P = a I + b A + c A A,  X <- P X
// Every product is C = U V' on 16-bit matrix instructions with 32-bit accuracy: a value is held as two fp16 planes
// (hi + lo, 22 bits, times a power of two that its bound allows: |X|, |A|, |P| have bounds that the coefficients set), and
// hi hi + hi lo + lo hi are accumulated in fp32.  The dropped lo lo is 2^-24 of the product.  Three fp16 products run at
// a third of the dense 2.5 PFLOP/s; fp32 matrix instructions stop at 0.16.
// All matrices of a call share the launches (one per product), their tiles side by side in the grid; A and P are symmetric,
// only the tiles on and above the diagonal are computed and the others mirrored.
#include "common.h"

namespace {

typedef _Float16 h16;
typedef __attribute__((ext_vector_type(8))) _Float16 h16x8;
typedef __attribute__((ext_vector_type(4))) _Float16 h16x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;

constexpr int PAD = 64;          // matrices are padded with zeros to multiples of this
constexpr int CHUNK = 4096;      // elements of one partial sum of squares
constexpr int NOPS = 32;         // matrices of one launch (their descriptions are kernel arguments: at most 4 KB)
constexpr int64_t MAXGRID = 1LL << 31;
constexpr float SX = 16384.f;    // |X| <= 3.9: fp16 ends at 65504
constexpr float SA = 4096.f;     // |A| <= 15.9
constexpr float SP = 1024.f;     // |P| <= 63

__host__ __device__ inline int64_t up64(int64_t v) { return (v + PAD - 1) / PAD * PAD; }

__device__ __forceinline__ void split(float v, h16& hi, h16& lo) {
    hi = (h16)v;
    lo = (h16)(v - (float)hi);
}

// One group of equal matrices, `stride` bytes apart in the workspace.
struct Mat {
    const void* g;   // sources, dense
    float* buf;      // momentum (NULL: orthogonalise g itself)
    char* ws;        // workspace of the first
    int64_t stride;
    int rows, cols;
    int first;       // first workgroup of this launch that works on the group
};

struct Mats {
    Mat mat[NOPS];
    int count;
    // momentum: u = mu buf + (1 - mu) g, buf before u; nesterov: u = mu buf + (1 - mu) g once more
    float mu;
    int nesterov;
    float eps;
};

// Byte offsets in one matrix's workspace: the scale, the partial sums, two X (each [m][n] and [n][m], hi plane then lo
// plane), A, P.
struct Lay {
    int64_t mp, np, scale, part, nparts, xm[2], xt[2], a, p, bytes;
};

__host__ __device__ inline Lay lay_of(int64_t rows, int64_t cols) {
    Lay l;
    l.mp = up64(rows < cols ? rows : cols);
    l.np = up64(rows < cols ? cols : rows);
    l.nparts = (rows * cols + CHUNK - 1) / CHUNK;
    int64_t at = 256;
    l.scale = 0;
    l.part = at;
    at += (l.nparts * 8 + 255) / 256 * 256;
    const int64_t x = l.mp * l.np * 4, sq = l.mp * l.mp * 4;
    for (int k = 0; k < 2; ++k) {
        l.xm[k] = at;
        at += x;
        l.xt[k] = at;
        at += x;
    }
    l.a = at;
    at += sq;
    l.p = at;
    at += sq;
    l.bytes = at;
    return l;
}

// the group that workgroup `id` works on (first[] ascends)
template <typename S>
__device__ __forceinline__ int group_of(const S& s, int id) {
    int lo = 0, hi = s.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (s.mat[mid].first <= id) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

template <typename T>
__device__ __forceinline__ float source(const Mats& s, const T* g, const float* buf, int64_t i) {
    const float v = (float)g[i];
    if (!buf) return v;
    const float m = buf[i];
    return s.nesterov ? fmaf(s.mu, m, (1.f - s.mu) * v) : m;
}

// ---- momentum and the partial sums of squares (doubles: no square of a finite fp32 leaves their range) ------------------
template <typename T>
__global__ void __launch_bounds__(256) ortho_norm_k(const Mats s) {
    __shared__ double red[4];
    const Mat& q = s.mat[group_of(s, blockIdx.x)];
    const int64_t size = (int64_t)q.rows * q.cols, nparts = (size + CHUNK - 1) / CHUNK;
    const int64_t local = blockIdx.x - q.first, b = local / nparts, c = local % nparts;
    const T* g = (const T*)q.g + b * size;
    float* buf = q.buf ? q.buf + b * size : nullptr;
    const int64_t end = (c + 1) * CHUNK < size ? (c + 1) * CHUNK : size;
    double sum = 0.;
    for (int64_t i = c * CHUNK + threadIdx.x; i < end; i += 256) {
        if (buf) buf[i] = fmaf(s.mu, buf[i], (1.f - s.mu) * (float)g[i]);
        const float u = source(s, g, buf, i);
        sum += (double)u * (double)u;
    }
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        char* ws = q.ws + b * q.stride;
        ((double*)(ws + 256))[c] = red[0] + red[1] + red[2] + red[3];
    }
}

// SX / max(|u|, eps) of each matrix, the partial sums in their order; not finite: NaN, so that the whole matrix says so
__global__ void __launch_bounds__(256) ortho_scale_k(const Mats s) {
    __shared__ double red[4];
    const Mat& q = s.mat[group_of(s, blockIdx.x)];
    const int64_t size = (int64_t)q.rows * q.cols, nparts = (size + CHUNK - 1) / CHUNK;
    char* ws = q.ws + (int64_t)(blockIdx.x - q.first) * q.stride;
    double sum = 0.;
    for (int64_t i = threadIdx.x; i < nparts; i += 256) sum += ((const double*)(ws + 256))[i];
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        const double n = sqrt(red[0] + red[1] + red[2] + red[3]);
        *(float*)ws = n < 1e300 ? (float)((double)SX / (n > (double)s.eps ? n : (double)s.eps)) : __builtin_nanf("");
    }
}

// ---- the scaled source as two planes, [rows][cols] and [cols][rows], padded with zeros ---------------------------------
template <typename T>
__global__ void __launch_bounds__(256) ortho_pack_k(const Mats s) {
    __shared__ float tile[64][65];
    const Mat& q = s.mat[group_of(s, blockIdx.x)];
    const int rp = (int)up64(q.rows), cp = (int)up64(q.cols);
    const int tr = rp / 64, tc = cp / 64;
    const int64_t local = blockIdx.x - q.first, b = local / ((int64_t)tr * tc);
    const int t = (int)(local % ((int64_t)tr * tc)), r0 = t / tc * 64, c0 = t % tc * 64;
    const int64_t size = (int64_t)q.rows * q.cols;
    const T* g = (const T*)q.g + b * size;
    const float* buf = q.buf ? q.buf + b * size : nullptr;
    char* ws = q.ws + b * q.stride;
    const float scale = *(const float*)ws;
    for (int k = threadIdx.x; k < 64 * 64; k += 256) {
        const int r = k >> 6, c = k & 63;
        const bool in = r0 + r < q.rows && c0 + c < q.cols;
        tile[r][c] = in ? scale * source(s, g, buf, (int64_t)(r0 + r) * q.cols + c0 + c) : 0.f;
    }
    __syncthreads();
    const Lay l = lay_of(q.rows, q.cols);
    const bool wide = q.rows <= q.cols;
    h16* nat = (h16*)(ws + (wide ? l.xm[0] : l.xt[0]));
    h16* tra = (h16*)(ws + (wide ? l.xt[0] : l.xm[0]));
    const int64_t plane = l.mp * l.np;
    for (int k = threadIdx.x; k < 64 * 8; k += 256) {
        const int r = k >> 3, c = (k & 7) * 8;
        h16x8 hi, lo, thi, tlo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            h16 x, y;
            split(tile[r][c + e], x, y);
            hi[e] = x;
            lo[e] = y;
            split(tile[c + e][r], x, y);
            thi[e] = x;
            tlo[e] = y;
        }
        const int64_t at = (int64_t)(r0 + r) * cp + c0 + c, ta = (int64_t)(c0 + r) * rp + r0 + c;
        *(h16x8*)(nat + at) = hi;
        *(h16x8*)(nat + plane + at) = lo;
        *(h16x8*)(tra + ta) = thi;
        *(h16x8*)(tra + plane + ta) = tlo;
    }
}

// ---- products ----------------------------------------------------------------------------------------------------------
enum Kind { GRAM = 0, POLY = 1, APPLY = 2, RESULT = 3 };

struct Op {
    char* ws;        // of the group's first matrix
    int64_t stride;
    void* out;       // RESULT
    int rows, cols;  // of the source
    int first, tiles;  // first workgroup, workgroups per matrix
    int kind, cur;     // cur: which X holds the iterate
};

struct Ops {
    Op mat[NOPS];
    int count;
    float a, b, c;
    float decay, step;  // RESULT onto parameters: p = decay p - step_of(rows, cols) X
    int update;         // 0: out = X; 1: the parameters; 2, 3: the step scaled by the shape, see step_of
};

__device__ __forceinline__ float step_of(const Ops& s, int rows, int cols) {
    const float r = (float)rows, c = (float)cols;
    return s.update == 2 ? s.step * sqrtf(fmaxf(1.f, r / c)) : s.update == 3 ? s.step * 0.2f * sqrtf(fmaxf(r, c)) : s.step;
}

// an address that is the same in every lane, in scalar registers
__device__ __forceinline__ const char* scalar(const char* p) {
    const uint64_t v = (uint64_t)p;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)v), hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32));
    return (const char*)(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_from(const char* p) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)scalar(p), 0, 0xffffffffu, 0x00020000);
}

// LDS-DMA of stage `step` into `base`: a wave's instruction j covers 1 KB = 16 rows of plane j / (T / 64)
template <int T, int PER>
__device__ __forceinline__ void ortho_issue(char* base, int step, int wave, __amdgpu_buffer_rsrc_t ru, __amdgpu_buffer_rsrc_t rul,
                                            __amdgpu_buffer_rsrc_t rv, __amdgpu_buffer_rsrc_t rvl, const unsigned (&off)[PER]) {
    constexpr int PP = T / 64;
#pragma unroll
    for (int j = 0; j < PER; ++j)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(j / PP == 0 ? ru : j / PP == 1 ? rul : j / PP == 2 ? rv : rvl,
                                                 (__attribute__((address_space(3))) void*)(base + (4 * j + wave) * 1024), 16, off[j], step * 64, 0,
                                                 0);
}

// Tile T x T of C = U V', four waves of T/2 x T/2.  U [M][K], V [N][K], each a hi plane and a lo plane; K % 32 == 0.  Stages of
// 32 k (64 bytes a row) go to LDS by DMA, chunk c of row r at position c ^ ((r >> 2) & 3): the 16 rows that a fragment read
// touches at a time then lie in different banks.
template <int T, int NST>
__global__ void __launch_bounds__(256, T == 128 ? 2 : 4) ortho_gemm_k(const Ops s, int dtype) {
    constexpr int F = T / 64;                     // 32 x 32 fragments of a wave, each way
    constexpr int PLANE = T * 64, STAGE = 4 * PLANE;  // bytes: U hi, U lo, V hi, V lo
    constexpr int PER = STAGE / 4096;             // DMA instructions per wave and stage
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const Op& q = s.mat[group_of(s, blockIdx.x)];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave >> 1, wn = wave & 1;
    // (divisions run on vector registers: say that the results are the wave's, or every use of an address loops over lanes)
    const int b = __builtin_amdgcn_readfirstlane((int)(blockIdx.x - q.first) / q.tiles);
    int t = (int)(blockIdx.x - q.first) - b * q.tiles;
    const Lay l = lay_of(q.rows, q.cols);
    char* ws = q.ws + b * q.stride;
    const int mp = (int)l.mp, np = (int)l.np;
    // operands
    const bool sym = q.kind <= POLY;
    const char *u, *v;
    int M, N, K;
    if (q.kind == GRAM) {
        u = v = ws + (q.cur ? l.xm[1] : l.xm[0]);
        M = N = mp;
        K = np;
    } else if (q.kind == POLY) {
        u = v = ws + l.a;
        M = N = K = mp;
    } else {
        u = ws + l.p;
        v = ws + (q.cur ? l.xt[1] : l.xt[0]);
        M = K = mp;
        N = np;
    }
    int ti, tj;
    if (sym) {  // tiles on and above the diagonal, row by row
        int left = (M + T - 1) / T;
        ti = 0;
        while (t >= left) {
            t -= left--;
            ++ti;
        }
        tj = ti + t;
    } else {
        const int tm = (M + T - 1) / T;
        tj = __builtin_amdgcn_readfirstlane(t / tm);
        ti = t - tj * tm;
    }
    const int i0 = ti * T, j0 = tj * T;
    // ---- staging: a wave's instruction j covers 1 KB of the stage = 16 rows of one plane
    const unsigned kb = (unsigned)K * 2;
    unsigned off[PER];
    const int rsub = lane >> 2, pos = lane & 3;
    const __amdgpu_buffer_rsrc_t ru = rows_from(u + (int64_t)i0 * kb);
    const __amdgpu_buffer_rsrc_t rul = rows_from(u + ((int64_t)M + i0) * kb);
    const __amdgpu_buffer_rsrc_t rv = rows_from(v + (int64_t)j0 * kb);
    const __amdgpu_buffer_rsrc_t rvl = rows_from(v + ((int64_t)N + j0) * kb);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int piece = 4 * j + wave, pl = piece / (T / 16), row = piece % (T / 16) * 16 + rsub;
        // rows past the matrix (T = 128 over an odd number of 64s): the last row again, their results are not stored
        const int lim = pl < 2 ? M - i0 : N - j0;
        off[j] = (unsigned)(row < lim ? row : lim - 1) * kb + (unsigned)((pos ^ ((row >> 2) & 3)) * 16);
    }
    f32x16 acc[F][F];
#pragma unroll
    for (int x = 0; x < F; ++x)
#pragma unroll
        for (int y = 0; y < F; ++y)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[x][y][r] = 0.f;
    const int nk = K / 32;
#pragma unroll
    for (int k = 0; k < NST - 1; ++k)
        if (k < nk) ortho_issue<T, PER>(lds + k * STAGE, k, wave, ru, rul, rv, rvl, off);
    for (int k = 0; k < nk; ++k) {
        // this wave's share of stage k has arrived and its reads of the stage before are done ...
        if (k + NST - 1 < nk + 1)
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NST - 2) * PER) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        // ... and everyone's
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (k + NST - 1 < nk)
            ortho_issue<T, PER>(lds + (k + NST - 1) % NST * STAGE, k + NST - 1, wave, ru, rul, rv, rvl, off);
        const char* base = lds + k % NST * STAGE;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            h16x8 uh[F], ul[F], vh[F], vl[F];
            const int ch = h * 2 + (lane >> 5);
#pragma unroll
            for (int x = 0; x < F; ++x) {
                const int ra = wm * (T / 2) + x * 32 + (lane & 31), rb = wn * (T / 2) + x * 32 + (lane & 31);
                const int pa = ra * 64 + ((ch ^ ((ra >> 2) & 3)) << 4), pb = rb * 64 + ((ch ^ ((rb >> 2) & 3)) << 4);
                uh[x] = *(const h16x8*)(base + pa);
                ul[x] = *(const h16x8*)(base + PLANE + pa);
                vh[x] = *(const h16x8*)(base + 2 * PLANE + pb);
                vl[x] = *(const h16x8*)(base + 3 * PLANE + pb);
            }
#pragma unroll
            for (int x = 0; x < F; ++x)
#pragma unroll
                for (int y = 0; y < F; ++y) acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(uh[x], vl[y], acc[x][y], 0, 0, 0);
#pragma unroll
            for (int x = 0; x < F; ++x)
#pragma unroll
                for (int y = 0; y < F; ++y) acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ul[x], vh[y], acc[x][y], 0, 0, 0);
#pragma unroll
            for (int x = 0; x < F; ++x)
#pragma unroll
                for (int y = 0; y < F; ++y) acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(uh[x], vh[y], acc[x][y], 0, 0, 0);
        }
    }
    // ---- results: lane holds column lane & 31, rows 8 (r / 4) + 4 (lane >> 5) + r % 4 of each 32 x 32 block
    const int64_t sq = (int64_t)mp * mp, xp = (int64_t)mp * np;
#pragma unroll
    for (int x = 0; x < F; ++x) {
#pragma unroll
        for (int y = 0; y < F; ++y) {
            const int ib = i0 + wm * (T / 2) + x * 32, j = j0 + wn * (T / 2) + y * 32 + (lane & 31);
            if (ib >= M || j >= N) continue;  // (both go by whole blocks of 32)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
                const int i = ib + 8 * r4 + 4 * (lane >> 5);
                float o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = acc[x][y][r4 * 4 + e];
                if (q.kind == RESULT) {
                    const bool wide = q.rows <= q.cols;
                    const float inv = 1.f / (SP * SX);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int row = wide ? i + e : j, col = wide ? j : i + e;
                        if (row >= q.rows || col >= q.cols) continue;
                        const int64_t at = ((int64_t)b * q.rows + row) * q.cols + col;
                        const float val = o[e] * inv;
                        if (s.update == 0) {
                            if (dtype == GAN_F32) ((float*)q.out)[at] = val;
                            else ((bf16*)q.out)[at] = (bf16)val;
                        } else {
                            float* p = (float*)q.out + at;
                            *p = fmaf(-step_of(s, q.rows, q.cols), val, s.decay * *p);
                        }
                    }
                    continue;
                }
                h16 *dn, *dt;        // [i][j] and [j][i]
                int64_t plane, ldn, ldt;
                if (q.kind == APPLY) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[e] *= 1.f / SP;
                    dn = (h16*)(ws + (q.cur ? l.xm[0] : l.xm[1]));
                    dt = (h16*)(ws + (q.cur ? l.xt[0] : l.xt[1]));
                    plane = xp;
                    ldn = np;
                    ldt = mp;
                } else {
                    if (q.kind == GRAM) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[e] *= SA / (SX * SX);
                    } else {
                        const h16* A = (const h16*)(ws + l.a);
                        const h16x4 ah = *(const h16x4*)(A + (int64_t)j * mp + i), al = *(const h16x4*)(A + sq + (int64_t)j * mp + i);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float av = ((float)ah[e] + (float)al[e]) * (SP / SA);
                            o[e] = fmaf(s.c * (SP / (SA * SA)), o[e], s.b * av) + (i + e == j ? s.a * SP : 0.f);
                        }
                    }
                    dn = dt = (h16*)(ws + (q.kind == GRAM ? l.a : l.p));
                    plane = sq;
                    ldn = ldt = mp;
                }
                h16x4 hi, lo;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    h16 p, w;
                    split(o[e], p, w);
                    hi[e] = p;
                    lo[e] = w;
                    dn[(int64_t)(i + e) * ldn + j] = p;
                    dn[plane + (int64_t)(i + e) * ldn + j] = w;
                }
                if (!sym || ti != tj) {
                    *(h16x4*)(dt + (int64_t)j * ldt + i) = hi;
                    *(h16x4*)(dt + plane + (int64_t)j * ldt + i) = lo;
                }
            }
        }
    }
}

// One product of every matrix, one launch.
int products(const gan_matrix* mats, int n, int kind, int cur, Ops& s, char* ws, int dtype, hipStream_t st) {
    constexpr int T = 64, NST = 2;
    int64_t blocks = 0;
    s.count = n;
    for (int k = 0; k < n; ++k) {
        const gan_matrix& g = mats[k];
        const Lay l = lay_of(g.rows, g.cols);
        Op& q = s.mat[k];
        q.ws = ws;
        q.stride = l.bytes;
        q.out = g.out;
        q.rows = (int)g.rows;
        q.cols = (int)g.cols;
        q.kind = kind;
        q.cur = cur;
        const int64_t tm = (l.mp + T - 1) / T, tn = (l.np + T - 1) / T;
        q.tiles = (int)(kind <= POLY ? tm * (tm + 1) / 2 : tm * tn);
        q.first = (int)blocks;
        blocks += (int64_t)q.tiles * g.batch;
        ws += l.bytes * g.batch;
    }
    hipLaunchKernelGGL((ortho_gemm_k<T, NST>), dim3((unsigned)blocks), dim3(256), NST * 4 * T * 64, st, s, dtype);
    GAN_CHECK_LAUNCH("orthogonalize(product)");
    return GAN_OK;
}

// The largest factor that a singular value can have grown to after each step, from 1: extremes of x |a + b x^2 + c x^4| on [0, r].
bool bounded(int steps, float a, float b, float c) {
    double r = 1.0;
    for (int k = 0; k < steps; ++k) {
        auto f = [&](double x) { return fabs(x * (a + b * x * x + c * x * x * x * x)); };
        auto p = [&](double x) { return fabs(a + b * x * x + c * x * x * x * x); };
        double top = f(r), poly = p(0.) > p(r) ? p(0.) : p(r);
        // f' = a + 3 b y + 5 c y^2 (y = x^2), p' = 2 x (b + 2 c y)
        const double disc = 9. * b * b - 20. * (double)a * c;
        double ys[3] = {-1., -1., -1.};
        if (c != 0.f) {
            if (disc >= 0.) {
                ys[0] = (-3. * b + sqrt(disc)) / (10. * c);
                ys[1] = (-3. * b - sqrt(disc)) / (10. * c);
            }
            ys[2] = -b / (2. * c);
        } else if (b != 0.f) {
            ys[0] = -(double)a / (3. * b);
        }
        for (double y : ys)
            if (y > 0. && y < r * r) {
                top = f(sqrt(y)) > top ? f(sqrt(y)) : top;
                poly = p(sqrt(y)) > poly ? p(sqrt(y)) : poly;
            }
        if (!(top <= 3.5) || !(poly <= 60.)) return false;  // (NaN too)
        r = top > 1e-3 ? top : 1e-3;
    }
    return true;
}

int64_t total_bytes(const gan_matrix* mats, int count) {
    int64_t n = 0;
    for (int k = 0; k < count; ++k) {
        const gan_matrix& g = mats[k];
        if (g.rows < 1 || g.cols < 1 || g.batch < 0 || g.rows > (1 << 20) || g.cols > (1 << 20) || g.batch > (1 << 30)) return -1;
        if (g.rows * g.cols > (1LL << 32) || (g.rows < g.cols ? g.rows : g.cols) > 32768) return -1;
        const int64_t one = lay_of(g.rows, g.cols).bytes;
        if (g.batch && one > (1LL << 60) / g.batch) return -1;
        n += one * g.batch;
        if (n > (1LL << 60)) return -1;
    }
    return n;
}

// The three launches in front of the products: momentum and norms, scales, planes.
template <typename T>
int pack(const gan_matrix* mats, int n, char* ws, Mats& s, hipStream_t st) {
    int64_t first[3][NOPS + 1] = {};
    s.count = n;
    for (int k = 0; k < n; ++k) {
        const gan_matrix& g = mats[k];
        const Lay l = lay_of(g.rows, g.cols);
        Mat& q = s.mat[k];
        q.g = g.g;
        q.buf = g.buf;
        q.ws = ws;
        q.stride = l.bytes;
        q.rows = (int)g.rows;
        q.cols = (int)g.cols;
        ws += l.bytes * g.batch;
        const int64_t per[3] = {l.nparts, 1, l.mp / 64 * (l.np / 64)};
        for (int j = 0; j < 3; ++j) first[j][k + 1] = first[j][k] + per[j] * g.batch;
    }
    for (int j = 0; j < 3; ++j) {
        for (int k = 0; k < n; ++k) s.mat[k].first = (int)first[j][k];
        const dim3 grid((unsigned)first[j][n]), block(256);
        if (j == 0) hipLaunchKernelGGL((ortho_norm_k<T>), grid, block, 0, st, s);
        else if (j == 1) hipLaunchKernelGGL(ortho_scale_k, grid, block, 0, st, s);
        else hipLaunchKernelGGL((ortho_pack_k<T>), grid, block, 0, st, s);
        GAN_CHECK_LAUNCH("orthogonalize(source)");
    }
    return GAN_OK;
}

int run_all(const char* what, const gan_matrix* all, int count, int steps, Mats& s, Ops& o, int dtype, char* ws, int64_t bytes, hipStream_t st) {
    GAN_CHECK_ARG(count >= 0 && (count == 0 || all), "%s: null list", what);
    GAN_CHECK_ARG(steps >= 1 && steps <= 100, "%s: 1 to 100 steps, got %d", what, steps);
    GAN_CHECK_ARG(s.eps > 0.f && s.eps < 1e30f, "%s: eps must be positive, got %g", what, (double)s.eps);
    GAN_CHECK_ARG(bounded(steps, o.a, o.b, o.c), "%s: with coefficients %g %g %g a singular value can grow beyond 3.5", what, (double)o.a,
                  (double)o.b, (double)o.c);
    const int64_t need = total_bytes(all, count);
    GAN_CHECK_ARG(need >= 0, "%s: a matrix has a size that is not supported (1 to 2^20 either way, the smaller at most 32768)", what);
    GAN_CHECK_ARG(need == 0 || (ws && bytes >= need), "%s: workspace of %lld bytes wanted, %lld given", what, (long long)need,
                  (long long)(ws ? bytes : 0));
    GAN_CHECK_ARG(((uintptr_t)ws % 256) == 0, "%s: workspace must be 256-byte aligned", what);
    for (int k = 0; k < count; ++k) {
        const gan_matrix& g = all[k];
        GAN_CHECK_ARG(!g.batch || (g.g && g.out && (!o.update || g.buf)), "%s: null pointer", what);
        const Lay l = lay_of(g.rows, g.cols);
        const int64_t tiles = l.mp / 64 * (l.np / 64);
        GAN_CHECK_ARG(g.batch <= MAXGRID / NOPS / (tiles > l.nparts ? tiles : l.nparts), "%s: %lld matrices of %lld x %lld are too many for one call",
                      what, (long long)g.batch, (long long)g.rows, (long long)g.cols);
    }
    gan_matrix some[NOPS];
    char* at = ws;
    for (int from = 0; from < count;) {
        int n = 0;
        int64_t used = 0;
        while (from < count && n < NOPS) {
            const gan_matrix& g = all[from++];
            if (!g.batch) continue;
            some[n++] = g;
            used += lay_of(g.rows, g.cols).bytes * g.batch;
        }
        if (!n) break;
        int rc = dtype == GAN_F32 ? pack<float>(some, n, at, s, st) : pack<bf16>(some, n, at, s, st);
        if (rc) return rc;
        for (int k = 0; k < steps; ++k) {
            if ((rc = products(some, n, GRAM, k & 1, o, at, dtype, st))) return rc;
            if ((rc = products(some, n, POLY, k & 1, o, at, dtype, st))) return rc;
            if ((rc = products(some, n, k + 1 < steps ? APPLY : RESULT, k & 1, o, at, dtype, st))) return rc;
        }
        at += used;
    }
    return GAN_OK;
}

}  // namespace

extern "C" int64_t gan_orthogonalize_workspace(const gan_matrix* mats, int count) {
    if (count < 0 || (count && !mats)) return -1;
    return total_bytes(mats, count);
}

extern "C" int gan_orthogonalize(const gan_matrix* mats, int count, int steps, float a, float b, float c, float eps, int dtype, void* ws,
                                 int64_t ws_bytes, gan_stream_t stream) {
    GAN_CHECK_ARG(dtype == GAN_F32 || dtype == GAN_BF16, "orthogonalize: bad dtype %d", dtype);
    for (int k = 0; mats && k < count; ++k) GAN_CHECK_ARG(!mats[k].buf, "orthogonalize: matrix %d has a momentum buffer", k);
    Mats s = {};
    Ops o = {};
    s.eps = eps;
    o.a = a;
    o.b = b;
    o.c = c;
    return run_all("orthogonalize", mats, count, steps, s, o, dtype, (char*)ws, ws_bytes, (hipStream_t)stream);
}

extern "C" int gan_muon_step(const gan_matrix* mats, int count, float lr, float momentum, int nesterov, float weight_decay, int scaling, int steps,
                             float a, float b, float c, float eps, void* ws, int64_t ws_bytes, gan_stream_t stream) {
    GAN_CHECK_ARG(lr >= 0.f && momentum >= 0.f && momentum < 1.f && weight_decay >= 0.f,
                  "muon_step: bad hyper-parameters (lr %g, momentum %g, weight_decay %g)", (double)lr, (double)momentum, (double)weight_decay);
    GAN_CHECK_ARG(scaling >= 0 && scaling <= 2, "muon_step: bad scaling %d", scaling);
    Mats s = {};
    Ops o = {};
    s.eps = eps;
    s.mu = momentum;
    s.nesterov = nesterov;
    o.a = a;
    o.b = b;
    o.c = c;
    o.update = 1 + scaling;
    o.decay = 1.f - lr * weight_decay;
    o.step = lr;
    return run_all("muon_step", mats, count, steps, s, o, GAN_F32, (char*)ws, ws_bytes, (hipStream_t)stream);
}
