// Newton-Schulz orthogonalisation of matrices and the optimiser step built on it (gfx950).
//   X = G / max(|G|, eps) (Frobenius norm; X is m x n with m <= n, a tall G is worked on as its transpose), then `steps` times
//   A = X X',  P = a I + b A + c A A,  X <- P X
// Every product is C = U V' on 16-bit matrix instructions with 32-bit accuracy: a value is held as two fp16 planes
// (hi + lo, 22 bits, times a power of two that its bound allows: |X|, |A|, |P| have bounds that the coefficients set), and
// hi hi + hi lo + lo hi are accumulated in fp32.  The dropped lo lo is 2^-24 of the product.  (22 bits end where the lo half falls into
// fp16's subnormals: entries of X below 1.5e-5 of the norm are held to 2e-12 of it, of A to 7e-12, of P to 2e-9.  Rows of 1e-4 of the
// others' size come out to 8e-6 of their own, of 1e-6 to 8e-4; the whole of the matrix is within 2e-6 all the same, and a scale of
// its own for every row would cost a pass over X a step.)  Three fp16 products cost a third
// of the fp16 rate, and fp32 matrix instructions run at an eighth of it (1.18 PFLOP/s and 0.154 for large products).
// Measured: P X of 2048 x 8192 in 166 us = 1.24 PFLOP/s of fp16 (0.41 of fp32 accuracy), A = X X' of it in 116 us (0.94; half
// of A is computed), A A in 37 (0.74: 136 tiles for 256 CUs); five iterations 1290 to 1460 us by the clock that
// the card holds, of 512 x 4608 170 to 190.  Large products are
// bound by the matrix instructions, those of a few hundred rows by their latency: 8 to 10 us a launch, 3 of them matrix
// instructions, the others the way of the first requests through the caches and the end of the workgroup.
// All matrices of a call share the launches (one per product), their tiles side by side in the grid; A and P are symmetric,
// only the tiles on and above the diagonal are computed and the others mirrored.
#include <type_traits>
#include <utility>

#include "common.h"

namespace {

typedef _Float16 h16;
typedef __attribute__((ext_vector_type(8))) _Float16 h16x8;
typedef __attribute__((ext_vector_type(4))) _Float16 h16x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;

constexpr int PAD = 64;          // matrices are padded with zeros to multiples of this
constexpr int MAXPARTS = 512;    // partial sums of squares of a matrix
constexpr int NOPS = 32;         // matrices of one launch (their descriptions are kernel arguments: at most 4 KB)
// Workgroups of a launch stay below these (work items are counted in 32 bits: 256 in a workgroup of the general path, 1024 in LDS)
constexpr int64_t MAXBLOCKS = 1LL << 24, MAXSMALL = 1LL << 22;
constexpr float SX = 16384.f;    // |X| <= 3.9: fp16 ends at 65504
constexpr float SA = 4096.f;     // |A| <= 15.9
constexpr float SP = 16.f;       // |P| and products of two of them <= 4000

__host__ __device__ inline int64_t up64(int64_t v) { return (v + PAD - 1) / PAD * PAD; }

__device__ __forceinline__ void split(float v, h16& hi, h16& lo) {
    asm("" : "+v"(v));  // (an fp32 value: a product fused into one of the conversions and rounded in front of the other gives halves that do not fit)
    hi = (h16)v;
    lo = (h16)(v - (float)hi);
}

// A matrix in the workspace: of every 32 columns of a row the hi halves, then the lo halves, 128 bytes together -- a line of the
// caches, which a product's step of 32 k takes as a whole (with the planes apart it would fetch every line twice).
__device__ __forceinline__ int64_t hi_at(int64_t row, int col, int64_t ld) { return row * 2 * ld + (col >> 5) * 64 + (col & 31); }
constexpr int LO = 32;  // the lo half, from the hi half

// eight values, the first in a column that is a multiple of eight
__device__ __forceinline__ void store_planes(h16* to, const float (&o)[8]) {
    h16x8 hi, lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        h16 p, w;
        split(o[e], p, w);
        hi[e] = p;
        lo[e] = w;
    }
    *(h16x8*)to = hi;
    *(h16x8*)(to + LO) = lo;
}

// elements of one partial sum of squares
__host__ __device__ inline int64_t chunk_of(int64_t size) {
    const int64_t c = (size + MAXPARTS - 1) / MAXPARTS;
    return c < 4096 ? 4096 : (c + 1023) / 1024 * 1024;
}
__host__ __device__ inline int64_t parts_of(int64_t size) { return (size + chunk_of(size) - 1) / chunk_of(size); }

// One group of equal matrices, `stride` bytes apart in the workspace.
struct Mat {
    const void* g;   // sources, dense
    float* buf;      // momentum (NULL: orthogonalise g itself)
    char* ws;        // workspace of the first
    int64_t stride;
    int64_t x;       // offset of X
    int rows, cols;
};

// momentum: u = mu buf + (1 - mu) g, buf before u; nesterov: u = mu buf + (1 - mu) g once more
struct Source {
    float mu, eps;
    int nesterov;
    float growth;  // what the steps can multiply X by at most (1 at least)
};

struct Mats {
    int count;
    Source from;
    int first[NOPS];  // each group's first workgroup
    Mat mat[NOPS];
};

// Byte offsets in one matrix's workspace: the partial sums, 1 / lift (256 bytes), two X (m x n), five symmetric m x m, the slices' tiles of a product that is cut.  All multiples of 256.
enum { A0, A1, P0, P1, Q0, SQUARES };
constexpr int LIFT_AT = MAXPARTS * 8;
struct Lay {
    int64_t mp, np, nparts, x[2], sq[SQUARES], join, bytes;
    int cut;
};

// What a product of `tiles` T x T tiles over `steps` steps of 32 k takes, in us, every tile's k in `cut` slices: a CU holds one, two
// or five workgroups (T = 256, 128, 64) at a time, a step of all of them takes as long as measured (2.45; 0.42 alone, 0.62 each where
// two share the CU; 0.19 and 0.2), a round begins and ends in 5 to 9 us, and slices are written and read again at 5 TB/s by one
// more launch.
double cost_of(int T, int64_t tiles, int cut, int64_t steps) {
    const int hold = T == 256 ? 1 : T == 128 ? 2 : 5;
    const double alone = T == 256 ? 2.45 : T == 128 ? 0.42 : 0.19, each = T == 128 ? 0.62 : 0.2, ends = T == 64 ? 5. : 9.;
    const int64_t wgs = tiles * cut, on_cu = ceil_div64(wgs % (256 * hold), 256);
    const double n = (double)ceil_div64(steps, cut);
    auto round = [&](int64_t p) { return p ? n * (p == 1 ? alone : (double)p * each) + ends : 0.; };
    return (double)(wgs / (256 * hold)) * round(hold) + round(on_cu) + (cut > 1 ? 4. + (double)wgs * T * T * 8e-6 / 5. : 0.);
}

int64_t tiles_of(int64_t M, int64_t N, bool sym, int T) {
    const int64_t tm = (M + T - 1) / T, tn = (N + T - 1) / T;
    return sym ? tm * (tm + 1) / 2 : tm * tn;
}

// The same with the best tile, C of M x N over K (cut: as it stands).
double least_cost(int64_t M, int64_t N, int64_t K, bool sym, int64_t batch, int cut) {
    double least = 1e30;
    for (int T = 64; T <= 256; T *= 2) {
        const double c = cost_of(T, tiles_of(M, N, sym, T) * batch, cut, K / 32);
        if (c < least) least = c;
    }
    return least;
}

// Slices of A = X X' (a long k, few tiles), at least eight steps each, by the group alone (the workspace goes by it).
int cut_of(int64_t mp, int64_t np, int64_t batch) {
    int best = 1;
    double least = 1e30;
    for (int T = 64; T <= 256; T *= 2) {
        const int64_t tiles = tiles_of(mp, mp, true, T), steps = np / 32;
        for (int64_t cut = 1; cut == 1 || (cut <= 256 / tiles && cut <= steps / 8); ++cut) {
            const double c = cost_of(T, tiles * batch, (int)cut, steps);
            if (c < least) {
                least = c;
                best = (int)cut;
            }
        }
    }
    const int64_t steps = np / 32, each = ceil_div64(steps, best);
    return (int)ceil_div64(steps, each);
}

Lay lay_of(const gan_matrix& g) {
    const int64_t rows = g.rows, cols = g.cols;
    Lay l;
    l.mp = up64(rows < cols ? rows : cols);
    l.np = up64(rows < cols ? cols : rows);
    l.nparts = parts_of(rows * cols);
    int64_t at = LIFT_AT + 256;
    const int64_t x = l.mp * l.np * 4, sq = l.mp * l.mp * 4;
    for (int k = 0; k < 2; ++k) {
        l.x[k] = at;
        at += x;
    }
    for (int k = 0; k < SQUARES; ++k) {
        l.sq[k] = at;
        at += sq;
    }
    l.join = at;
    l.cut = cut_of(l.mp, l.np, g.batch);
    const int64_t t = (l.mp + 255) / 256 * 4;  // in whole tiles of the largest size
    if (l.cut > 1) at += l.cut * t * (t + 4) / 2 * 4096 * 4;
    l.bytes = at;
    return l;
}

// The most workgroups that one of these matrices takes in a launch: a product's tiles of 64, or, where sums are cut in slices, up to
// 4096 tiles of slices, or every 32 x 32 block on and above the diagonal, in whole tiles, for the launch that joins them.
int64_t blocks_of(const Lay& l) {
    const int64_t t = l.mp / 64, tiles = t * (l.np / 64);
    return (tiles > l.nparts ? tiles : l.nparts) + (l.cut > 1 ? 4096 + 2 * (t + 3) * (t + 7) : 0);
}

// the group that workgroup `id` works on (first[] ascends)
template <typename S>
__device__ __forceinline__ int group_of(const S& s, int id) {
    int lo = 0, hi = s.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (s.first[mid] <= id) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// what is orthogonalised, of gradient g and momentum m
__device__ __forceinline__ float update_of(const Source& s, float g, float m) { return s.nesterov ? fmaf(s.mu, m, (1.f - s.mu) * g) : m; }

// ---- momentum and the partial sums of squares (doubles: no square of a finite fp32 leaves their range) ------------------
template <typename T>
__global__ void __launch_bounds__(256) ortho_norm_k(const Mats s) {
    __shared__ double red[4];
    const int group = group_of(s, blockIdx.x);
    const Mat q = s.mat[group];
    const int64_t size = (int64_t)q.rows * q.cols, chunk = chunk_of(size), nparts = parts_of(size);
    const int local = (int)blockIdx.x - s.first[group], b = local / (int)nparts, c = local - b * (int)nparts;
    const T* __restrict__ g = (const T*)q.g + b * size;
    float* __restrict__ buf = q.buf ? q.buf + b * size : nullptr;
    const int64_t end = (c + 1) * chunk < size ? (c + 1) * chunk : size;
    double sum = 0.;
    for (int64_t i0 = c * chunk; i0 < end; i0 += 1024) {  // four elements a thread and round, all requested at once
        const int64_t i = i0 + threadIdx.x * 4;
        float v[4], m[4];
        if (i + 4 <= end) {
            T t[4];
            __builtin_memcpy(t, g + i, sizeof(t));
            if (buf) __builtin_memcpy(m, buf + i, sizeof(m));
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (float)t[e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = i + e < end ? (float)g[i + e] : 0.f;
                m[e] = buf && i + e < end ? buf[i + e] : 0.f;
            }
        }
        if (buf) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                m[e] = fmaf(s.from.mu, m[e], (1.f - s.from.mu) * v[e]);
                v[e] = update_of(s.from, v[e], m[e]);
            }
            if (i + 4 <= end) {
                __builtin_memcpy(buf + i, m, sizeof(m));
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (i + e < end) buf[i + e] = m[e];
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) sum += (double)v[e] * (double)v[e];
    }
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) ((double*)(q.ws + b * q.stride))[c] = red[0] + red[1] + red[2] + red[3];
}

// SX / max(|u|, eps) times the lift.  A matrix of a norm far below eps stays small through all steps; its halves would fall into fp16's
// subnormals (a norm of 1e-5 eps: four digits), so X is held a power of two higher, as far as `growth` leaves room: 1 for a norm of
// eps and more.  (One for all steps: an entry of average size then is held to 2^-38 growth sqrt(m n) of it, 2.7e-6 for 512 x 4608 in
// five.)  A is held as it is (as small as it then is, P is a I and little else).  Not finite: NaN, so that the whole matrix says so.
__device__ __forceinline__ float scale_of(double norm, const Source& s, float& lift) {
    lift = 1.f;
    if (!(norm < 1e300)) return __builtin_nanf("");
    double scale = (double)SX / (norm > (double)s.eps ? norm : (double)s.eps);
    int up;
    frexp(norm / (double)s.eps * (double)s.growth, &up);
    if (norm > 0. && up < 0) {
        for (up = up < -100 ? -100 : up; up < 0 && ldexp(scale, -up) > 1e37; ++up) {}  // (fp32)
        lift = (float)ldexp(1., -up);
        scale = ldexp(scale, -up);
    }
    return (float)scale;
}

// Of the partial sums in their order, every workgroup for itself and all the same
__device__ __forceinline__ float scale_of(const double* part, int nparts, const Source& s, float& lift) {
    __shared__ double red[4];
    double sum = 0.;
    for (int i = threadIdx.x; i < nparts; i += 256) sum += part[i];
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
    __syncthreads();
    return scale_of(sqrt(red[0] + red[1] + red[2] + red[3]), s, lift);
}

// ---- the scaled source as m x n, padded with zeros (a tall source transposed) --------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256) ortho_pack_k(const Mats s) {
    __shared__ float tile[64][65];
    const int group = group_of(s, blockIdx.x);
    const Mat q = s.mat[group];
    const int rp = (int)up64(q.rows), cp = (int)up64(q.cols);
    const int tr = rp / 64, tc = cp / 64;
    const int64_t local = blockIdx.x - s.first[group], b = local / ((int64_t)tr * tc);
    const int t = (int)(local % ((int64_t)tr * tc)), r0 = t / tc * 64, c0 = t % tc * 64;
    const int64_t size = (int64_t)q.rows * q.cols;
    const T* g = (const T*)q.g + b * size;
    const float* buf = q.buf ? q.buf + b * size : nullptr;
    char* ws = q.ws + b * q.stride;
    float v[16], m[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        const int r = r0 + k * 4 + (threadIdx.x >> 6), c = c0 + (threadIdx.x & 63);
        const bool in = r < q.rows && c < q.cols;
        const int64_t at = in ? (int64_t)r * q.cols + c : 0;  // always loaded, cleared afterwards
        v[k] = (float)g[at];
        if (buf) m[k] = buf[at];
        if (!in) v[k] = m[k] = 0.f;
    }
    float lift;
    const float scale = scale_of((const double*)ws, (int)parts_of(size), s.from, lift);
    if (t == 0 && threadIdx.x == 0) *(float*)(ws + LIFT_AT) = 1.f / lift;
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        const int r = k * 4 + (threadIdx.x >> 6), c = threadIdx.x & 63;
        const bool in = r0 + r < q.rows && c0 + c < q.cols;
        tile[r][c] = in ? scale * (buf ? update_of(s.from, v[k], m[k]) : v[k]) : 0.f;
    }
    __syncthreads();
    h16* to = (h16*)(ws + q.x);
    const bool wide = q.rows <= q.cols;
    for (int k = threadIdx.x; k < 64 * 8; k += 256) {
        const int r = k >> 3, c = (k & 7) * 8;
        float o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = wide ? tile[r][c + e] : tile[c + e][r];
        store_planes(to + (wide ? hi_at(r0 + r, c0 + c, cp) : hi_at(c0 + r, r0 + c, rp)), o);
    }
}

// ---- products ----------------------------------------------------------------------------------------------------------
enum Kind { SCALED, POLY, CHAIN, RESULT };  // gain U V'; c U V' + b aux + a I; c U V' + b aux + a aux2; the call's result

// C = U V' (or U V) of one group of equal matrices
struct Op {
    char* ws;          // of the group's first matrix
    int64_t stride;
    void* out;         // RESULT
    unsigned u, v;     // operands, result, POLY's and CHAIN's further terms, slices: in 256 bytes from ws
    unsigned to, aux, aux2, join;
    int M, N, K;       // padded
    int apply;         // C = U V with V [K][N] as it lies, not transposed; else C is symmetric: tiles on and above the diagonal
    int rows, cols;    // of the source
    int tiles;         // per matrix
    int cut, steps;    // slices of k, steps of 32 k in each but the last
    int kind;
    int lifts;         // how often X is a factor of the product without being one of the result
    float gain;        // of the product; P and what CHAIN adds have the scale SP, POLY's A has SA
};

// the polynomial, and what becomes of the result
struct Rule {
    float a, b, c;
    float decay, step;  // RESULT onto parameters: p = decay p - step_of(rows, cols) X
    int update;         // 0: out = X; 1: the parameters; 2, 3: the step scaled by the shape, see step_of
};

struct Ops {
    int count;
    Rule rule;
    int first[NOPS + 1];  // each group's first workgroup, and behind the last
    Op mat[NOPS];
};

__device__ __forceinline__ float step_of(const Rule& s, int rows, int cols) {
    const float r = (float)rows, c = (float)cols;
    return s.update == 2 ? s.step * sqrtf(fmaxf(1.f, r / c)) : s.update == 3 ? s.step * 0.2f * sqrtf(fmaxf(r, c)) : s.step;
}

// Tile t of the tiles on and above the diagonal of n x n: strips of four tile rows, down the columns of each.  A run of sixteen
// tiles then reads eight row blocks of the operand, not seventeen as along a row: what a die's cache has to bring in from the
// memory side, at 8 TB/s over all of them, bounds these products.
__device__ __forceinline__ int2 tile_of(int t, int n) {
    int top = 0, h = n < 4 ? n : 4;
    for (;;) {
        const int all = h * (h + 1) / 2 + h * (n - top - h);
        if (t < all) break;
        t -= all;
        top += 4;
        h = n - top < 4 ? n - top : 4;
    }
    int c = 0;
    for (; c < h; ++c) {  // the triangle on the diagonal
        if (t <= c) return make_int2(top + t, top + c);
        t -= c + 1;
    }
    c = t / h;
    return make_int2(top + t - c * h, top + h + c);
}

// A wave's 32 x 32 block of a product at (i0, j0), as accumulated: lane holds column lane & 31, rows 8 (r / 4) + 4 (lane >> 5) +
// r % 4.  It goes through `t` (the wave's own LDS) once, so that the block and, of a symmetric result, its transpose (mirror: where
// that is another block's place) are stored 16 bytes a lane.
constexpr int TLD = 36;  // floats a row: 16-byte rows, and columns of eight spread over the banks
constexpr int TBYTES = 32 * TLD * 4;

// eight values of a row of the result, `left` of them inside it: stored, or taken off the parameters there
template <typename T>
__device__ __forceinline__ void store_result(const Rule& rule, T* to, float (&o)[8], int left, float step) {
    if (left >= 8) {
        if (rule.update) {
            T old[8];
            __builtin_memcpy(old, to, sizeof(old));
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = fmaf(-step, o[e], rule.decay * (float)old[e]);
        }
        T r[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = (T)o[e];
        __builtin_memcpy(to, r, sizeof(r));
    } else {
#pragma unroll
        for (int e = 0; e < 7; ++e)
            if (e < left) to[e] = (T)(rule.update ? fmaf(-step, o[e], rule.decay * (float)to[e]) : o[e]);
    }
}

// 1 / lift where the product has it too often.  (A scalar load: the kernels' vector loads are counted, and none is waited for early.)
__device__ __forceinline__ float unlift_of(const Op& q, const char* ws) {
    return q.lifts ? *(const __attribute__((address_space(4))) float*)(uintptr_t)(ws + LIFT_AT) : 1.f;
}

__device__ __forceinline__ void finish(const Ops& s, const Op& q, char* ws, float unlift, int b, int i0, int j0, f32x16& acc, bool mirror, int dtype,
                                       float* t) {
    const int lane = threadIdx.x & 63;
    // the values first, where the accumulators hold them: no branch or load stands between the trips through LDS
    if (q.kind == POLY || q.kind == CHAIN) {  // (what is added is symmetric: its rows for the columns held here)
        const int64_t at = hi_at(j0 + (lane & 31), i0 + 4 * (lane >> 5), q.N);
        const h16* A = (const h16*)(ws + (int64_t)q.aux * 256) + at;
        h16x4 ah[4], al[4], ph[4], pl[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            ah[r] = *(const h16x4*)(A + 8 * r);
            al[r] = *(const h16x4*)(A + LO + 8 * r);
        }
        if (q.kind == CHAIN) {
            const h16* P = (const h16*)(ws + (int64_t)q.aux2 * 256) + at;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                ph[r] = *(const h16x4*)(P + 8 * r);
                pl[r] = *(const h16x4*)(P + LO + 8 * r);
            }
        }
        const float c = s.rule.c * q.gain, bb = s.rule.b * (q.kind == POLY ? SP / SA : 1.f);
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[r] = fmaf((float)ah[r >> 2][r & 3], bb, fmaf((float)al[r >> 2][r & 3], bb, acc[r] * c));
        if (q.kind == CHAIN) {
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[r] = fmaf((float)ph[r >> 2][r & 3], s.rule.a, fmaf((float)pl[r >> 2][r & 3], s.rule.a, acc[r]));
        } else if (i0 == j0) {
            const int on = (lane & 31) - 4 * (lane >> 5);  // the row of the diagonal
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[r] += on == 8 * (r >> 2) + (r & 3) ? s.rule.a * SP : 0.f;
        }
    } else {
        const float gain = (q.kind == SCALED ? q.gain : 1.f / (SP * SX)) * unlift * (q.lifts == 2 ? unlift : 1.f);
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[r] *= gain;
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int r = 0; r < 16; ++r) t[(8 * (r >> 2) + 4 * (lane >> 5) + (r & 3)) * TLD + (lane & 31)] = acc[r];
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    const int a = lane >> 2, c = (lane & 3) * 8;  // eight values a lane: columns c ... of rows a and a + 16, or the other way round
    float o[2][8], x[2][8];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            o[h][e] = t[(h * 16 + a) * TLD + c + e];
            x[h][e] = t[(c + e) * TLD + h * 16 + a];
        }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the next block may overwrite them)
    if (q.kind == RESULT) {
        const bool wide = q.rows <= q.cols;  // a tall result is the transpose of the block
        const float step = s.rule.update ? step_of(s.rule, q.rows, q.cols) : 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int row = (wide ? i0 : j0) + h * 16 + a, col = (wide ? j0 : i0) + c;
            const int left = row < q.rows ? q.cols - col : 0;
            const int64_t at = ((int64_t)b * q.rows + row) * q.cols + col;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = wide ? o[h][e] : x[h][e];
            if (dtype == GAN_F32) store_result(s.rule, (float*)q.out + at, v, left, step);
            else store_result(s.rule, (bf16*)q.out + at, v, left, step);
        }
        return;
    }
    h16* to = (h16*)(ws + (int64_t)q.to * 256);
#pragma unroll
    for (int h = 0; h < 2; ++h) store_planes(to + hi_at(i0 + h * 16 + a, j0 + c, q.N), o[h]);
    if (mirror) {
#pragma unroll
        for (int h = 0; h < 2; ++h) store_planes(to + hi_at(j0 + h * 16 + a, i0 + c, q.N), x[h]);
    }
}

// An address that is the same in every lane, in scalar registers.  (Five wait states lie between a vector instruction's write of a
// scalar register and its use by a memory instruction; the compiler does not see the one in ortho_issue.)
__device__ __forceinline__ const char* scalar(const char* p) {
    const uint64_t v = (uint64_t)p;
    uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)v), hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32));
    asm volatile("s_nop 4" : "+s"(lo), "+s"(hi));
    return (const char*)(((uint64_t)hi << 32) | lo);
}

// One LDS-DMA instruction: instruction j of the waves covers WAVES pieces of 1 KB of the stage at `base`, T / 8 pieces of U and then
// T / 8 of V.  u, v: the operands' first bytes, at: the stage's bytes from there.  Written out, since the compiler would wait for
// every request on its way in front of any transposing read of LDS (it cannot tell the stages apart); stage_arrived() waits for
// what is needed.
template <int T, int WAVES>
__device__ __forceinline__ void ortho_issue(char* base, unsigned at_u, unsigned at_v, int wave, const char* u, const char* v, const unsigned* off, int j) {
    typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
    const bool of_u = WAVES * j < T / 8;
    const uint64_t from = (uint64_t)(of_u ? u : v);
    const u32x4 rsrc = {(unsigned)from, (unsigned)(from >> 32), 0xffffffffu, 0x00020000u};
    const unsigned to = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)(base + (WAVES * j + wave) * 1024);
    const unsigned at = of_u ? at_u : at_v;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(to), "v"(off[j]), "s"(rsrc), "s"(at) : "m0");
}

// Of four rows (k) of sixteen elements, lane i of sixteen brings the four at (row i / 4, columns 4 (i % 4) ...) and takes column
// i of the four rows.
__device__ __forceinline__ h16x4 read_transposed(const char* p) {
    typedef __attribute__((ext_vector_type(4))) short s16x4;
    return __builtin_bit_cast(h16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
}

// The fragments of 16 k of a wave's tile, from the stage at `base`: rows m0 ... of U, n0 ... of V
template <int FM, int FN>
struct Frags {
    static constexpr int READS = 2 * (FM + FN), PRODUCTS = 3 * FM * FN;
    h16x8 u[2][FM], v[2][FN];  // hi, lo
    // APPLY: V's stage is [32 k][T], 16 columns of it at a time turned round on the way
    template <int T, bool APPLY>
    __device__ __forceinline__ void read(const char* base, int m0, int n0, int half, int lane, int r) {
        const bool of_u = r < 2 * FM;
        const int f = (of_u ? r : r - 2 * FM) >> 1, pl = r & 1;
        if (APPLY && !of_u) {
            const int row = half * 16 + (lane >> 5) * 8 + ((lane & 15) >> 2);
            const int chunk = (n0 / 32 + f) * 8 + pl * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
            const char* p = base + T * 128 + row * (T * 4) + ((chunk ^ ((row & 3) << 2)) << 4) + (lane & 1) * 8;
            const h16x4 a = read_transposed(p), b = read_transposed(p + 4 * (T * 4));
            v[pl][f] = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
            return;
        }
        const int row = (of_u ? m0 : n0) + f * 32 + (lane & 31), chunk = pl * 4 + half * 2 + (lane >> 5);
        const h16x8 got = *(const h16x8*)(base + (of_u ? 0 : T * 128) + row * 128 + ((chunk ^ ((row >> 1) & 7)) << 4));
        if (of_u) u[pl][f] = got;
        else v[pl][f] = got;
    }
    // hi lo, lo hi, hi hi, each over all of the wave's blocks (a block's accumulator then rests between two products); a wave with
    // one block only has an accumulator for each of the three
    static constexpr int NACC = FM * FN == 1 ? 3 : 1;
    __device__ __forceinline__ void multiply(f32x16 (&acc)[NACC][FM][FN], int i) const {
        const int pass = i / (FM * FN), x = i % (FM * FN) / FN, y = i % FN, a = NACC == 3 ? pass : 0;
        acc[a][x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(u[pass == 1][x], v[pass == 0][y], acc[a][x][y], 0, 0, 0);
    }
};

// Waits until a stage is in LDS for everyone and everyone's earlier reads are done: this wave's last N requests may still be on
// their way if all of them are (`full`: later stages), else none.
template <int N>
__device__ __forceinline__ void stage_arrived(bool full) {
    if (full)
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
    else
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Tile T x T of C = U V' or U V: four waves of T/2 x T/2 each, or (T = 256) eight of 128 x 64.  KG = 2: two such sets of four, each
// with one half of every stage; their sums are added at the end.  That is for grids of a workgroup a CU at most, where a lone
// wave on its SIMD would have nothing beside it while it waits.
// U [M][K], V [N][K] or [K][N]; K % 32 == 0.  Stages of 32 k go to LDS by DMA.  Of a matrix with k along its rows a stage holds a
// line (128 bytes: hi, lo) a row, chunk c of row r at position c ^ ((r >> 1) & 7): the 16 rows that a fragment read touches at a
// time then lie in different banks.  Of [K][N] it holds 32 rows of T, chunk c of row r at c ^ 4 (r & 3): the four rows of 64
// bytes that a transposing read touches fill the banks.
template <int T, int NST, int KG>
__global__ void __launch_bounds__(T == 256 ? 512 : 256 * KG, T == 64 ? 4 : 2) ortho_gemm_k(const Ops s, int dtype) {
    constexpr int SET = T == 256 ? 8 : 4, WAVES = SET * KG, WN = SET / 2;  // a set's waves: 2 x WN
    constexpr int FM = T / 64, FN = T / 32 / WN;                   // 32 x 32 fragments of a wave
    constexpr int STAGE = 2 * T * 128;                             // bytes: U, V
    constexpr int PER = STAGE / 1024 / WAVES;                      // DMA instructions per wave and stage
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int group = group_of(s, blockIdx.x);
    const Op q = s.mat[group];  // (a copy: one batch of scalar loads)
    // Workgroups go round the eight dies, each with a cache of its own: of each group's, a die gets a run.  Tiles follow one
    // another along the rows of U, sharing their rows of V, and a slice's tiles lie together.
    const int all = s.first[group + 1] - s.first[group], local = (int)blockIdx.x - s.first[group];
    const int each = all >> 3, rest = all & 7, die = local & 7;
    const int id = die * each + (die < rest ? die : rest) + (local >> 3);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), in_set = wave % SET, kg = wave / SET,
              wm = in_set / WN, wn = in_set % WN;
    // (divisions run on vector registers: say that the results are the wave's, or every use of an address loops over lanes)
    const int per = q.tiles * q.cut;
    const int b = __builtin_amdgcn_readfirstlane(id / per);
    const int in_b = id - b * per;
    const int slice = __builtin_amdgcn_readfirstlane(in_b / q.tiles), tile = in_b - slice * q.tiles;
    char* ws = q.ws + b * q.stride;
    const float unlift = unlift_of(q, ws);  // (here, so that nobody waits for it at the end)
    const char *u = ws + (int64_t)q.u * 256, *v = ws + (int64_t)q.v * 256;
    const int M = q.M, N = q.N, K = q.K;
    int ti, tj;
    if (q.apply) {
        const int tm = (M + T - 1) / T;
        tj = __builtin_amdgcn_readfirstlane(tile / tm);
        ti = tile - tj * tm;
    } else {
        const int2 t = tile_of(tile, (M + T - 1) / T);
        ti = __builtin_amdgcn_readfirstlane(t.x);
        tj = __builtin_amdgcn_readfirstlane(t.y);
    }
    const int i0 = ti * T, j0 = tj * T;
    // ---- staging: a wave's instruction j covers 1 KB of the stage: eight rows with k along them, or part of one that runs along n
    const unsigned kb = (unsigned)K * 4, nb = (unsigned)N * 4, v_step = q.apply ? 32 * nb : 128;
    unsigned off[PER];
    const char* const pu = scalar(u + (int64_t)i0 * kb);
    const char* const pv = scalar(v + (q.apply ? (int64_t)j0 * 4 : (int64_t)j0 * kb));
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int piece = WAVES * j + wave;
        const bool of_u = piece < T / 8;
        const int at = (of_u ? piece : piece - T / 8) * 1024 + lane * 16;
        // rows (columns) past the matrix (T = 128 over an odd number of 64s): the last again, their results are not stored
        if (of_u || !q.apply) {
            const int row = at / 128, pos = at % 128 / 16, lim = of_u ? M - i0 : N - j0;
            off[j] = (unsigned)(row < lim ? row : lim - 1) * kb + (unsigned)((pos ^ ((row >> 1) & 7)) * 16);
        } else {
            const int row = at / (T * 4), pos = at % (T * 4) / 16, chunk = pos ^ ((row & 3) << 2), lim = (N - j0) / 4 - 1;
            off[j] = (unsigned)row * nb + (unsigned)(chunk < lim ? chunk : lim) * 16;
        }
    }
    using Fr = Frags<FM, FN>;
    f32x16 sums[Fr::NACC][FM][FN];
#pragma unroll
    for (int a = 0; a < Fr::NACC; ++a)
#pragma unroll
        for (int x = 0; x < FM; ++x)
#pragma unroll
            for (int y = 0; y < FN; ++y)
#pragma unroll
                for (int r = 0; r < 16; ++r) sums[a][x][y][r] = 0.f;
    const int k0 = slice * q.steps, nk = (K / 32 - k0 < q.steps ? K / 32 - k0 : q.steps);
    auto issue = [&](char* base, int step, int j) __attribute__((always_inline)) {
        ortho_issue<T, WAVES>(base, (unsigned)(k0 + step) * 128, (unsigned)(k0 + step) * v_step, wave, pu, pv, off, j);
    };
#pragma unroll
    for (int k = 0; k < NST; ++k)
        if (k < nk) {
#pragma unroll
            for (int j = 0; j < PER; ++j) issue(lds + k * STAGE, k, j);
        }
    // While the matrix instructions of one half of a stage (16 k) run, the other half's fragments are read and DMA is asked for,
    // a piece behind each: eight requests in a row would hold the wave at the address unit (64 bytes a clock for the CU) for as
    // long as a third of its products take.  The barrier lies between the halves, where the next stage has to be there and
    // nobody reads this one any more; its place is then filled with stage k + NST, half of the requests before and half after
    // the next half's turn.
    constexpr int HALF = PER / 2;
    const int m0 = wm * (T / 2), n0 = wn * (T / WN);
    auto walk = [&](auto apply) __attribute__((always_inline)) {
        constexpr bool APPLY = decltype(apply)::value;
        Fr f0, f1;
        if constexpr (KG == 2) {
            // this set's half of the next stage is read, and the stage after the last asked for, while its half of this one runs
            auto step = [&](int k, Fr& now, Fr& then, bool more) __attribute__((always_inline)) {
                stage_arrived<(NST - 2) * PER>(k + NST - 1 < nk);
#pragma unroll
                for (int i = 0; i < Fr::PRODUCTS; ++i) {
                    now.multiply(sums, i);
#pragma unroll
                    for (int r = 0; r < Fr::READS; ++r)
                        if (r * Fr::PRODUCTS / (2 * Fr::READS) == i)
                            then.template read<T, APPLY>(lds + (k + 1) % NST * STAGE, m0, n0, kg, lane, r);
                    if (more) {
#pragma unroll
                        for (int j = 0; j < PER; ++j)
                            if ((j + 1) * Fr::PRODUCTS / PER - 1 == i) issue(lds + k % NST * STAGE, k + NST, j);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            stage_arrived<(NST - 1) * PER>(nk >= NST);
#pragma unroll
            for (int r = 0; r < Fr::READS; ++r) f0.template read<T, APPLY>(lds, m0, n0, kg, lane, r);
            int k = 0;
            for (; k + 1 + NST < nk; k += 2) {
                step(k, f0, f1, true);
                step(k + 1, f1, f0, true);
            }
            for (; k + 2 < nk; k += 2) {
                step(k, f0, f1, k + NST < nk);
                step(k + 1, f1, f0, k + 1 + NST < nk);
            }
            if (k + 1 < nk) step(k, f0, f1, k + NST < nk);
            const Fr& tail = k + 1 < nk ? f1 : f0;
#pragma unroll
            for (int i = 0; i < Fr::PRODUCTS; ++i) tail.multiply(sums, i);
            return;
        }
        stage_arrived<(NST - 1) * PER>(nk >= NST);
#pragma unroll
        for (int r = 0; r < Fr::READS; ++r) f0.template read<T, APPLY>(lds, m0, n0, 0, lane, r);
        auto step = [&](int k, bool late, bool more) __attribute__((always_inline)) {
            char *here = lds + k % NST * STAGE, *last = lds + (k + NST - 1) % NST * STAGE, *next = lds + (k + 1) % NST * STAGE;
#pragma unroll
            for (int i = 0; i < Fr::PRODUCTS; ++i) {
                f0.multiply(sums, i);
#pragma unroll
                for (int r = 0; r < Fr::READS; ++r)
                    if (r * Fr::PRODUCTS / (2 * Fr::READS) == i) f1.template read<T, APPLY>(here, m0, n0, 1, lane, r);
                if (late) {
#pragma unroll
                    for (int j = 0; j < HALF; ++j)
                        if ((j + 1) * Fr::PRODUCTS / HALF - 1 == i) issue(last, k - 1 + NST, HALF + j);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            stage_arrived<(NST - 2) * PER>(k + NST - 1 < nk);  // stages k + 2 ... k + NST - 1 behind it
#pragma unroll
            for (int i = 0; i < Fr::PRODUCTS; ++i) {
                f1.multiply(sums, i);
#pragma unroll
                for (int r = 0; r < Fr::READS; ++r)
                    if (r * Fr::PRODUCTS / (2 * Fr::READS) == i) f0.template read<T, APPLY>(next, m0, n0, 0, lane, r);
                if (more) {
#pragma unroll
                    for (int j = 0; j < HALF; ++j)
                        if ((j + 1) * Fr::PRODUCTS / HALF - 1 == i) issue(here, k + NST, j);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        if (nk > 1) step(0, false, NST < nk);
        int k = 1;
        for (; k + NST < nk; ++k) step(k, true, true);
        for (; k + 1 < nk; ++k) step(k, k - 1 + NST < nk, false);
        const char* here = lds + (nk - 1) % NST * STAGE;
#pragma unroll
        for (int r = 0; r < Fr::READS; ++r) f1.template read<T, APPLY>(here, m0, n0, 1, lane, r);
#pragma unroll
        for (int i = 0; i < Fr::PRODUCTS; ++i) f0.multiply(sums, i);
#pragma unroll
        for (int i = 0; i < Fr::PRODUCTS; ++i) f1.multiply(sums, i);
    };
    if (q.apply) walk(std::true_type{});
    else walk(std::false_type{});
    f32x16(&acc)[FM][FN] = sums[0];
    if (Fr::NACC == 3) {
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[0][0][r] = sums[Fr::NACC - 1][0][0][r] + (acc[0][0][r] + sums[Fr::NACC / 2][0][0][r]);
    }
    // the blocks that this wave goes on with, in a row: all of the set's, or its set's share once the sets' sums are added
    constexpr int BLOCKS = FM * FN, KEEP = KG == 1 ? BLOCKS : (BLOCKS + 1) / 2;
    const int keep = kg * KEEP;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();  // (the stages are read: their LDS is free)
    if constexpr (KG == 2) {
        float4* x = (float4*)lds + in_set * BLOCKS * 256 + lane;
#pragma unroll
        for (int f = 0; f < BLOCKS; ++f)
            if (f / KEEP != kg) {  // the other set's
                const f32x16& o = acc[f / FN][f % FN];
#pragma unroll
                for (int r = 0; r < 4; ++r) x[(f * 4 + r) * 64] = make_float4(o[r * 4], o[r * 4 + 1], o[r * 4 + 2], o[r * 4 + 3]);
            }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
#pragma unroll
        for (int f = 0; f < BLOCKS; ++f)
            if (f / KEEP == kg) {
                f32x16& o = acc[f / FN][f % FN];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float4 v = x[(f * 4 + r) * 64];
                    o[r * 4] += v.x;
                    o[r * 4 + 1] += v.y;
                    o[r * 4 + 2] += v.z;
                    o[r * 4 + 3] += v.w;
                }
            }
    }
    float4* out = (float4*)(ws + (int64_t)q.join * 256) + ((int64_t)slice * q.tiles + tile) * (T * T / 4) + in_set * (T * T / 4 / SET) + lane;
    float* t = (float*)(lds + (KG == 1 ? 0 : SET * BLOCKS * 4096) + wave * TBYTES);
    // one block after another through the same code: unrolled, its instructions would be fetched for every block anew
#pragma unroll 1
    for (int f = keep; f < BLOCKS && f < keep + KEEP; ++f) {
        f32x16 one = acc[0][0];
#pragma unroll
        for (int k = 1; k < BLOCKS; ++k)
            if (f == k) one = acc[k / FN][k % FN];
        const int i = i0 + wm * (T / 2) + f / FN * 32, j = j0 + wn * (T / WN) + f % FN * 32;
        if (q.cut > 1) {  // this slice's sums, in the order that join_k reads them
#pragma unroll
            for (int r = 0; r < 4; ++r) out[(f * 4 + r) * 64] = make_float4(one[r * 4], one[r * 4 + 1], one[r * 4 + 2], one[r * 4 + 3]);
        } else if (i < M && j < N) {
            finish(s, q, ws, unlift, b, i, j, one, !q.apply && ti != tj, dtype, t);
        }
    }
}

// The slices of a product that was cut, added in their order; a 32 x 32 block a workgroup of one wave
template <int T>
__global__ void __launch_bounds__(64) ortho_join_k(const Ops s, int dtype) {
    constexpr int WAVES = T == 256 ? 8 : 4, WN = WAVES / 2, FN = T / 32 / WN, BLK = T * T / 1024;  // blocks of a tile
    __shared__ __attribute__((aligned(16))) float lds[TBYTES / 4];
    const int group = group_of(s, blockIdx.x);
    const Op q = s.mat[group];
    const int lane = threadIdx.x;
    const int local = (int)blockIdx.x - s.first[group], tile_b = local / BLK, b = tile_b / q.tiles, tile = tile_b - b * q.tiles;
    char* ws = q.ws + b * q.stride;
    const float unlift = unlift_of(q, ws);
    const int blk = local % BLK, wave = blk / (BLK / WAVES), frag = blk % (BLK / WAVES);
    const float4* in = (const float4*)(ws + (int64_t)q.join * 256) + (int64_t)tile * (T * T / 4) + blk * 256 + lane;
    const int64_t next = (int64_t)q.tiles * (T * T / 4);
    f32x16 acc;
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[r] = 0.f;
    constexpr int AHEAD = 8;  // slices requested at a time
    for (int c = 0; c < q.cut; c += AHEAD) {
        float4 v[AHEAD][4];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
#pragma unroll
            for (int r = 0; r < 4; ++r) v[k][r] = in[(c + k < q.cut ? c + k : c) * next + r * 64];
        __builtin_amdgcn_sched_barrier(0);  // (or the loads are moved to their uses, one wait each)
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const bool in_cut = c + k < q.cut;
                acc[r * 4] += in_cut ? v[k][r].x : 0.f;
                acc[r * 4 + 1] += in_cut ? v[k][r].y : 0.f;
                acc[r * 4 + 2] += in_cut ? v[k][r].z : 0.f;
                acc[r * 4 + 3] += in_cut ? v[k][r].w : 0.f;
            }
    }
    const int2 t = tile_of(tile, (q.M + T - 1) / T);
    const int i = t.x * T + (wave / WN) * (T / 2) + frag / FN * 32, j = t.y * T + (wave % WN) * (T / WN) + frag % FN * 32;
    if (i < q.M && j < q.N) finish(s, q, ws, unlift, b, i, j, acc, t.x != t.y, dtype, lds);
}

template <int T, int NST, int KG>
int launch_gemm(unsigned blocks, const Ops& s, int dtype, hipStream_t st) {
    constexpr int lds = NST * 2 * T * 128;
    // more than 64 KB of dynamic LDS needs the attribute (set on every call: it is per device, and cheap)
    if (lds > 64 * 1024 && hipFuncSetAttribute((const void*)ortho_gemm_k<T, NST, KG>, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) {
        gan_set_error("orthogonalize: cannot reserve %d bytes of LDS", lds);
        return GAN_ERR_LAUNCH;
    }
    hipLaunchKernelGGL((ortho_gemm_k<T, NST, KG>), dim3(blocks), dim3(T == 256 ? 512 : 256 * KG), lds, st, s, dtype);
    GAN_CHECK_LAUNCH("orthogonalize(product)");
    return GAN_OK;
}

// What a matrix does in the launches, one after another: stages of one or two iterations, each from A = X X' anew.
//   one:  P = poly(A);                                                     X <- P X
//   two:  P = poly(A), T = P A, A2 = P T (= X2 X2'), P2 = poly(A2), Q = P2 P;  X <- Q X
//   two, side by side:  P = poly(A) | T = P A, S = P P | A2 = T P, B = T S (= A2 P) | Q = a P + b B + c A2 B;  X <- Q X
// Two iterations at a time replace a product with X and one into it by three m x m ones: 6 m^2 n + 2 m^3 against
// 3 m^2 n + 5 m^3, which can pay from n = 2 m on.  Not more at a time: an error of A, 2^-22 of its largest singular value, weighs
// the more on the smallest ones the longer the iteration runs on A alone (error against 64 bits, 512 x 4608 with a spectrum that
// falls like 1 / i: 1.9e-6 step by step, 3.1e-6 like this, 7.8e-6 in stages of two and three, 1.7e-4 in one).  The first
// stage is a single iteration: the small values are smallest there.
// Side by side is a product more and a launch less: taken where two products of each matrix leave no CU with more than one tile,
// the launch then being as long as one (512 x 4608: 195 -> 184 us, 704 x 1500 187 -> 178; 1000 x 4000, which has more tiles, gains nothing).
// Up to 192 rows they are not taken, alone or in a list, where they leave more than fp32 products do (13 of 70 x 2589: 3.7e-6 in 143 us
// against 1.4e-6 in 163, fp32 products 1.6e-6; in lists 64 x 576 3.6e-6 against 1.2e-6, fp32 products 2.0e-6, and 171 x 340 2.2e-6
// against 1.0e-6, 1.6e-6; a discriminator's list takes 400 to 411 us instead of 393 for it).  Beyond that they have to gain a launch's time by
// the cost rule: else step by step it is, the more accurate way (300 x 700: 0.7e-6 in 122 us against 1.8e-6 in 121; 512 x 4608: 1.2e-6 in
// 193 us, taken are 1.6e-6 in 175).  Where several sizes share the launches, all of more than 192 rows go the same way as far as they
// can, whatever each would gain alone: a discriminator's step would take 485 us with some of its large matrices step by step; their errors
// are 0.4 to 1.2 times those of fp32 products, most at 193 to 256 rows (0.4 to 0.6 step by step).
bool two_at_a_time(const Lay& l, int64_t batch, bool beside, bool shared) {
    if (l.np < 2 * l.mp || l.mp <= 192) return false;
    if (shared) return true;
    const double gram = least_cost(l.mp, l.mp, l.np, true, batch, l.cut), apply = least_cost(l.mp, l.np, l.mp, false, batch, 1),
                 square = least_cost(l.mp, l.mp, l.mp, true, batch, 1);
    return gram + apply - (beside ? 2 : 3) * square >= 6.;
}

struct Walk {
    Lay l;
    bool pairs, beside;       // two iterations at a time; side by side
    int left, size, at, cur;  // iterations left, this stage's size, the next launch within it, the X that holds the iterate
    // one or two products
    int next(Op* q, int steps) {
        if (at == 0) size = pairs && left < steps && left >= 2 ? 2 : 1;
        int n = 0;
        auto sq = [&](int k) { return (unsigned)(l.sq[k] / 256); };
        auto mul = [&](int u, int v, int to, float gain, int kind = SCALED, int aux = 0, int aux2 = 0) {
            Op& o = q[n++];
            o.u = sq(u);
            o.v = sq(v);
            o.to = sq(to);
            o.aux = sq(aux);
            o.aux2 = sq(aux2);
            o.apply = 0;
            o.gain = gain;
            o.kind = kind;
            o.lifts = kind == RESULT ? 1 : 0;
            o.cut = 1;
            o.M = o.N = o.K = (int)l.mp;
        };
        const float poly = SP / (SA * SA);
        const int last = size == 1 ? 2 : beside ? 5 : 6;
        if (at == 0) {
            mul(0, 0, A0, SA / (SX * SX));
            q->lifts = 2;
            q->u = q->v = (unsigned)(l.x[cur] / 256);
            q->K = (int)l.np;
            q->cut = l.cut;
        } else if (at == last) {
            mul(size == 1 ? P0 : Q0, 0, 0, 1.f / SP, left == size ? RESULT : SCALED);
            q->v = (unsigned)(l.x[cur] / 256);
            q->to = (unsigned)(l.x[cur ^ 1] / 256);
            q->apply = 1;
            q->N = (int)l.np;
        } else if (at == 1) {
            mul(A0, A0, P0, poly, POLY, A0);
        } else if (at == 2) {
            mul(P0, A0, Q0, 1.f / SP);
            if (beside) mul(P0, P0, P1, 1.f / SP);
        } else if (at == 3) {
            mul(P0, Q0, A1, 1.f / SP);
            if (beside) mul(Q0, P1, A0, 1.f / SA);
        } else if (beside) {
            mul(A1, A0, Q0, 1.f / SA, CHAIN, A0, P0);
        } else if (at == 4) {
            mul(A1, A1, P1, poly, POLY, A1);
        } else {
            mul(P1, P0, Q0, 1.f / SP);
        }
        if (at++ == last) {
            left -= size;
            cur ^= 1;
            at = 0;
        }
        return n;
    }
};

// The next product of every matrix that has one left: one launch, and one more that joins slices where there are any.
int products(const gan_matrix* mats, Walk* walks, int n, int steps, Ops& s, char* ws, int dtype, hipStream_t st) {
    s.count = 0;
    bool sliced = false;
    int64_t batch[NOPS];
    for (int k = 0; k < n; ++k) {
        Walk& w = walks[k];
        for (int left = w.left ? w.next(s.mat + s.count, steps) : 0; left > 0; --left) {
            batch[s.count] = mats[k].batch;
            Op& q = s.mat[s.count++];
            q.ws = ws;
            q.stride = w.l.bytes;
            q.out = mats[k].out;
            q.rows = (int)mats[k].rows;
            q.cols = (int)mats[k].cols;
            q.join = (unsigned)(w.l.join / 256);
            q.steps = (int)ceil_div64(q.K / 32, q.cut);
            sliced |= q.cut > 1;
        }
        ws += w.l.bytes * mats[k].batch;
    }
    // long sums first: what starts last should end soon
    for (int k = 1; k < s.count; ++k)
        for (int j = k; j > 0 && s.mat[j].steps > s.mat[j - 1].steps; --j) {
            std::swap(s.mat[j], s.mat[j - 1]);
            std::swap(batch[j], batch[j - 1]);
        }
    // one tile size for the launch: the one that takes least, counted as if all its workgroups ran over the longest k
    int T = 64;
    double least = 1e30;
    for (int t = 64; t <= 256; t *= 2) {
        int64_t wgs = 0, longest = 0;
        for (int k = 0; k < s.count; ++k) {
            const Op& q = s.mat[k];
            wgs += tiles_of(q.M, q.N, !q.apply, t) * q.cut * batch[k];
            if (q.steps > longest) longest = q.steps;
        }
        const double c = cost_of(t, wgs, 1, longest);
        if (c < least) {
            least = c;
            T = t;
        }
    }
    int64_t blocks = 0;
    for (int k = 0; k < s.count; ++k) {
        Op& q = s.mat[k];
        q.tiles = (int)tiles_of(q.M, q.N, !q.apply, T);
        s.first[k] = (int)blocks;
        blocks += (int64_t)q.tiles * q.cut * batch[k];
    }
    s.first[s.count] = (int)blocks;
    // Where there is a workgroup a CU at most, a long ring of stages and two sets of waves (KG = 2) hide the waits: 116 us against 182
    // for A = X X' of 2048 x 8192.  Where there are more, those do, and short rings let more of them in: two of T = 128 a CU
    // (174 us against 184 for P X), five of T = 64 (14.3 us against 15.5 for 576 tiles of k = 512); up to two a CU of T = 64 keep the
    // long ring (five iterations of 1500 x 1500, 300 tiles: 405 us against 423 with two sets of waves and 480 with short rings).
    int rc;
    const unsigned grid = (unsigned)blocks;
    if (T == 256) rc = launch_gemm<256, 2, 1>(grid, s, dtype, st);
    else if (T == 128) rc = blocks > 256 ? launch_gemm<128, 2, 1>(grid, s, dtype, st) : launch_gemm<128, 4, 2>(grid, s, dtype, st);
    else if (blocks > 512) rc = launch_gemm<64, 2, 1>(grid, s, dtype, st);
    else rc = blocks > 256 ? launch_gemm<64, 4, 1>(grid, s, dtype, st) : launch_gemm<64, 4, 2>(grid, s, dtype, st);
    if (rc) return rc;
    if (!sliced) return GAN_OK;
    int64_t join = 0;
    int m = 0;
    for (int k = 0; k < s.count; ++k) {
        if (s.mat[k].cut == 1) continue;
        s.mat[m] = s.mat[k];
        s.first[m] = (int)join;
        join += (int64_t)s.mat[m++].tiles * batch[k] * (T * T / 1024);
    }
    s.count = m;
    if (T == 256) hipLaunchKernelGGL((ortho_join_k<256>), dim3((unsigned)join), dim3(64), 0, st, s, dtype);
    else if (T == 128) hipLaunchKernelGGL((ortho_join_k<128>), dim3((unsigned)join), dim3(64), 0, st, s, dtype);
    else hipLaunchKernelGGL((ortho_join_k<64>), dim3((unsigned)join), dim3(64), 0, st, s, dtype);
    GAN_CHECK_LAUNCH("orthogonalize(join)");
    return GAN_OK;
}

// ---- matrices that fit into LDS: one workgroup of sixteen waves each does everything, in one launch ---------------------------
// X lies there once, as [n][m]: P X reads it along the rows, A = X X' through transposing reads; A, then P, lie behind it, their
// blocks on and below the diagonal only (what lies above is read transposed).  A row is made of 128-byte lines, of 32 elements
// the hi and then the lo halves, and 16 bytes more: sixteen rows at one place, and four rows four apart over 64 bytes, then lie
// in different banks; neighbouring rows lie four apart (slot_of), so that a transposing read takes them in their order.  A
// product's results wait in registers (one or two 32 x 32 blocks a wave) until everyone has read the operands that they replace.
// The vector instructions around the products (halves, addresses) take as long as the products, and all of it is fetched cold
// once: little code, and addresses of one number a lane and constants.  Five iterations: 16 x 144 18 us, 128 x 128 39 us (a step
// 6.6 us, of which A, A A and P X take 1.3 + 1.5 + 1.8), 64 x 512 41 us where the launches of the general path (5 to 8 us each) took
// 100; 512 matrices of 64 x 512 102 us (320).
constexpr int SMALL_LDS = 160 * 1024 - 512;
constexpr int SMALL_BLOCKS = 32;                   // of 32 x 32, of X: two a wave
constexpr int SMALL_QUADS = SMALL_BLOCKS * 256 / 1024;  // a thread's groups of four source elements

struct SmallMat {
    const void* g;
    float* buf;
    void* out;
    int rows, cols;
};
struct Smalls {
    int count, steps;
    int first[NOPS];
    SmallMat mat[NOPS];
};

__host__ __device__ inline int up32(int v) { return (v + 31) & ~31; }

int small_bytes(int64_t rows, int64_t cols) {
    const int m = up32((int)(rows < cols ? rows : cols)), n = up32((int)(rows < cols ? cols : rows));
    return (m + n) * (m * 4 + 16);
}

bool is_small(const gan_matrix& g) {
    if (g.rows > 1024 || g.cols > 1024) return false;
    return up32((int)g.rows) * up32((int)g.cols) <= SMALL_BLOCKS * 1024 && small_bytes(g.rows, g.cols) <= SMALL_LDS;
}

// Where row `row` lies: of sixteen rows 4 a + b at place 4 b + a.
__device__ __forceinline__ int slot_of(int row) { return (row & ~15) | (row & 3) << 2 | ((row >> 2) & 3); }

// A matrix in LDS at byte `base` (a number, not a pointer: every address is then known to lie in LDS), and the lane's places in it
struct SmallView {
    unsigned base, pitch, row, col;
    __device__ __forceinline__ SmallView(unsigned b, int mp, int lane)
        : base(b), pitch(mp * 4 + 16), row(slot_of(lane & 31) * pitch + (lane >> 5) * 16),
          col(((lane >> 5) * 2 + (lane & 12)) * pitch + ((lane >> 4) & 1) * 32 + (lane & 3) * 8) {}
    template <typename V>
    static __device__ __forceinline__ __attribute__((address_space(3))) V& value(unsigned at) {
        return *(__attribute__((address_space(3))) V*)(uintptr_t)at;
    }
    // the 16 elements from column 16 kk of rows 32 blk ...: a lane row lane & 31 and eight of them
    __device__ __forceinline__ h16x8 along(int blk, int kk, int pl) const {
        return value<h16x8>(base + blk * 32 * pitch + kk / 2 * 128 + row + kk % 2 * 32 + pl * 64);
    }
    // the same of the transpose: places 0 4 8 12, 1 5 9 13 of the sixteen rows from 16 kk (lanes from 32 on: 2 ..., 3 ...)
    __device__ __forceinline__ h16x8 across(int blk, int kk, int pl) const {
        typedef __attribute__((ext_vector_type(4))) short s16x4;
        const unsigned p = base + kk * 16 * pitch + blk * 128 + col;
        const h16x4 a = __builtin_bit_cast(h16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(&value<s16x4>(p + pl * 64))),
                    b = __builtin_bit_cast(h16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(&value<s16x4>(p + pitch + pl * 64)));
        return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    // four values from column `col` (a multiple of four) on, of row `at`
    __device__ __forceinline__ void store(unsigned at, int col, const float (&v)[4]) const {
        h16x4 hi, lo;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            h16 x, y;
            split(v[e], x, y);
            hi[e] = x;
            lo[e] = y;
        }
        const unsigned to = at + (col >> 5) * 128 + (col & 31) * 2;
        value<h16x4>(to) = hi;
        value<h16x4>(to + 64) = lo;
    }
    // block (bi, bj) of a product, as accumulated: stored transposed
    __device__ __forceinline__ void store(int bi, int bj, const f32x16& a, float gain) const {
        const unsigned to = base + bj * 32 * pitch + bi * 128 + place();
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float v[4] = {gain * a[r * 4], gain * a[r * 4 + 1], gain * a[r * 4 + 2], gain * a[r * 4 + 3]};
            store(to, 8 * r, v);
        }
    }
    // of that block: the lane's column, its first row
    __device__ __forceinline__ unsigned place() const { return row - (threadIdx.x & 32) / 4; }
};

// A wave's products over the k from 32 from to 32 end: a block of rows `ub` of U by `vb` of V, or by U's own (B = 0), or by two
// blocks of V, vb and vb + 1 (B = 2).  TU, TV: k runs down the columns.  The next 16 are read while one is multiplied, with no
// branch in between (behind one, a wait would be for all reads).  A single block has an accumulator for hi hi and one for the
// others.
template <bool TU, bool TV, int B>
__device__ __forceinline__ void small_part(f32x16 (&acc)[2], const SmallView& U, int ub, const SmallView& V, int vb, int from, int end) {
    if (from >= end) return;
    struct Pieces {
        h16x8 u[2], v[2], w[2];
    } f[2];
    auto read = [&](Pieces& p, int kk) __attribute__((always_inline)) {
#pragma unroll
        for (int pl = 0; pl < 2; ++pl) {
            p.u[pl] = TU ? U.across(ub, kk, pl) : U.along(ub, kk, pl);
            if (B) p.v[pl] = TV ? V.across(vb, kk, pl) : V.along(vb, kk, pl);
            if (B == 2) p.w[pl] = V.along(vb + 1, kk, pl);
        }
    };
    auto multiply = [&](const Pieces& p) __attribute__((always_inline)) {
        const h16x8(&u)[2] = p.u, (&v)[2] = B ? p.v : p.u, (&w)[2] = p.w;
        if (B == 2) {
            acc[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(u[0], v[1], acc[0], 0, 0, 0);
            acc[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(u[0], w[1], acc[1], 0, 0, 0);
            acc[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(u[1], v[0], acc[0], 0, 0, 0);
            acc[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(u[1], w[0], acc[1], 0, 0, 0);
            acc[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(u[0], v[0], acc[0], 0, 0, 0);
            acc[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(u[0], w[0], acc[1], 0, 0, 0);
        } else {
            acc[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(u[0], v[1], acc[1], 0, 0, 0);
            acc[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(u[0], v[0], acc[0], 0, 0, 0);
            acc[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(u[1], v[0], acc[1], 0, 0, 0);
        }
    };
    read(f[0], 2 * from);
    int k = from;
#pragma unroll 1
    for (; k + 1 < end; ++k) {
        read(f[1], 2 * k + 1);
        multiply(f[0]);
        read(f[0], 2 * k + 2);
        multiply(f[1]);
    }
    read(f[1], 2 * k + 1);
    multiply(f[0]);
    multiply(f[1]);
}

__device__ __forceinline__ void clear(f32x16 (&acc)[2]) {
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[0][r] = acc[1][r] = 0.f;
}

template <typename T>
__global__ void __launch_bounds__(1024) ortho_small_k(const Smalls s, const Source h, const Rule o) {
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    __shared__ double red[16];
    const int group = group_of(s, blockIdx.x);
    const SmallMat q = s.mat[group];
    const int rows = q.rows, cols = q.cols, size = rows * cols;
    const int64_t b = (int)blockIdx.x - s.first[group];
    const bool wide = rows <= cols;
    const int m = wide ? rows : cols, n = wide ? cols : rows, mp = up32(m), np = up32(n);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    SmallView X((unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds, mp, lane), Q(X.base + np * X.pitch, mp, lane);
    // ---- source: momentum, norm, planes.  A thread has groups of four elements i ... i + 3 of a column j of X, neighbours in
    // memory beside each other's; zeros past the matrix.
    const T* g = (const T*)q.g + b * size;
    float* buf = q.buf ? q.buf + b * size : nullptr;
    auto element = [](auto* of, unsigned i) __attribute__((always_inline)) -> auto& {  // (32 bits of offset: one instruction less or four each)
        return *(decltype(of))((const char*)of + i * (unsigned)sizeof(*of));
    };
    const int fast = wide ? np : mp / 4, quads = mp * np / 4, slow0 = tid / fast, fast0 = tid - slow0 * fast, dslow = 1024 / fast,
              dfast = 1024 - dslow * fast;
    auto each = [&](auto&& f) __attribute__((always_inline)) {
        int a = slow0, c = fast0;
#pragma unroll
        for (int k = 0; k < SMALL_QUADS; ++k) {
            if (k * 1024 >= quads) break;
            f(k, wide ? c : a, 4 * (wide ? a : c));
            c += dfast;
            a += dslow;
            if (c >= fast) {
                c -= fast;
                ++a;
            }
        }
    };
    const unsigned di = wide ? cols : 1, dj = wide ? 1 : cols;
    float val[SMALL_QUADS][4];
    // (what is outside: the first element instead, cleared afterwards, so that no load stands behind a branch)
    each([&](int k, int j, int i) __attribute__((always_inline)) {
        const unsigned at = i * di + j * dj;
        const int in = j < n ? m - i : 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) val[k][e] = (float)element(g, e < in ? at + e * di : 0u);
    });
    if (buf) {
        float old[SMALL_QUADS][4];
        each([&](int k, int j, int i) __attribute__((always_inline)) {
            const unsigned at = i * di + j * dj;
            const int in = j < n ? m - i : 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) old[k][e] = element(buf, e < in ? at + e * di : 0u);
        });
        each([&](int k, int j, int i) __attribute__((always_inline)) {
            const unsigned at = i * di + j * dj;
            const int in = j < n ? m - i : 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float u = fmaf(h.mu, old[k][e], (1.f - h.mu) * val[k][e]);
                val[k][e] = update_of(h, val[k][e], u);
                if (e < in) element(buf, at + e * di) = u;
            }
        });
    }
    double sum = 0.;
    each([&](int k, int j, int i) __attribute__((always_inline)) {
        const int in = j < n ? m - i : 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            val[k][e] = e < in ? val[k][e] : 0.f;
            sum = fma((double)val[k][e], (double)val[k][e], sum);
        }
    });
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
    if (lane == 0) red[wave] = sum;
    __syncthreads();
    sum = 0.;
#pragma unroll
    for (int w = 0; w < 16; ++w) sum += red[w];
    const double norm = sqrt(sum);
    float lift;
    const float scale = scale_of(norm, h, lift);
    const float unlift = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, 1.f / lift)));
    each([&](int k, int j, int i) __attribute__((always_inline)) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = scale * val[k][e];
        if (k * 1024 + tid < quads) X.store(X.base + slot_of(j) * X.pitch, i, v);
    });
    __syncthreads();
    // ---- iterations; lane holds column lane & 31, rows 8 r + 4 (lane >> 5) ... + 3 of a block, which is stored transposed
    const int bm = mp / 32, bn = np / 32;
    int si = wave, sj = 0;  // of the blocks (si <= sj) of a symmetric product
    while (si > sj) si -= ++sj;
    const bool square = sj < bm;
    // Of P X two blocks with the same rows of P a wave where there are more of them than waves.  (Where they are not needed, pairs read
    // less of LDS but leave waves idle that hide what the others wait for: 128 x 128 3990 clocks alone, 4530 in pairs.)
    const bool pairs = bm * bn > 16;
    const int ai = wave % bm, aj = wave / bm * (pairs ? 2 : 1);
    const bool apply = aj < bn, two = pairs && aj + 1 < bn;
    f32x16 acc[2];
#pragma unroll 1
    for (int step = 0; step < s.steps; ++step) {
        // (sums of these are not kept from one step to the next: there are no registers for them)
        asm volatile("" : "+v"(X.row), "+v"(X.col), "+v"(Q.row), "+v"(Q.col));
        if (square) {
            clear(acc);
            if (si == sj) small_part<true, true, 0>(acc, X, si, X, sj, 0, bn);
            else small_part<true, true, 1>(acc, X, si, X, sj, 0, bn);
            acc[0] += acc[1];
            Q.store(si, sj, acc[0], SA / (SX * SX) * unlift * unlift);
        }
        __syncthreads();
        if (square) {
            clear(acc);
            const int below = si + 1, above = sj + 1, end = bm;
            if (si == sj) {
                small_part<false, false, 0>(acc, Q, si, Q, sj, 0, below);
                small_part<true, true, 0>(acc, Q, si, Q, sj, below, end);
            } else {
                small_part<false, false, 1>(acc, Q, si, Q, sj, 0, below);
                small_part<true, false, 1>(acc, Q, si, Q, sj, below, above);
                small_part<true, true, 1>(acc, Q, si, Q, sj, above, end);
            }
            acc[0] += acc[1];
            const unsigned A = Q.base + sj * 32 * Q.pitch + si * 128 + Q.place();
            const float cc = o.c * (SP / (SA * SA)), bb = o.b * (SP / SA);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const h16x4 ah = Q.value<h16x4>(A + 16 * r), al = Q.value<h16x4>(A + 16 * r + 64);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[0][r * 4 + e] = fmaf((float)ah[e], bb, fmaf((float)al[e], bb, acc[0][r * 4 + e] * cc));
            }
            if (si == sj) {
                const int on = (lane & 31) - 4 * (lane >> 5);  // the row of the diagonal
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[0][r] += on == 8 * (r >> 2) + (r & 3) ? o.a * SP : 0.f;
            }
        }
        __syncthreads();
        if (square) Q.store(si, sj, acc[0], 1.f);
        __syncthreads();
        if (apply) {
            clear(acc);
            const int below = ai + 1, end = bm;
            if (two) {
                small_part<false, false, 2>(acc, Q, ai, X, aj, 0, below);
                small_part<true, false, 2>(acc, Q, ai, X, aj, below, end);
            } else {
                small_part<false, false, 1>(acc, Q, ai, X, aj, 0, below);
                small_part<true, false, 1>(acc, Q, ai, X, aj, below, end);
                acc[0] += acc[1];
            }
        }
        if (step + 1 == s.steps) break;
        __syncthreads();
        if (apply) {
            X.store(ai, aj, acc[0], 1.f / SP);
            if (two) X.store(ai, aj + 1, acc[1], 1.f / SP);
        }
        __syncthreads();
    }
    if (!apply) return;
    const float shaped = o.update ? step_of(o, rows, cols) : 0.f;
    T* out = (T*)q.out + b * size;
#pragma unroll
    for (int z = 0; z < 2; ++z) {
        if (z && !two) break;
        const int i0 = ai * 32 + 4 * (lane >> 5), j = (aj + z) * 32 + (lane & 31), in = j < n ? m - i0 : 0;
        const unsigned at = i0 * di + j * dj;
        float old[16];
        if (o.update) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int e = 8 * (r >> 2) + (r & 3);
                old[r] = (float)element(out, e < in ? at + e * di : 0u);
            }
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int e = 8 * (r >> 2) + (r & 3);
            const float x = acc[z][r] * (1.f / (SP * SX) * unlift);
            if (e < in) element(out, at + e * di) = (T)(o.update ? fmaf(-shaped, x, o.decay * old[r]) : x);
        }
    }
}

template <typename T>
int run_small(const gan_matrix* mats, int n, int steps, const Source& h, const Rule& o, hipStream_t st) {
    Smalls s;
    int lds = 0, blocks = 0;
    s.count = n;
    s.steps = steps;
    for (int k = 0; k < n; ++k) {
        const gan_matrix& g = mats[k];
        s.mat[k] = SmallMat{g.g, g.buf, g.out, (int)g.rows, (int)g.cols};
        s.first[k] = blocks;
        blocks += (int)g.batch;
        const int need = small_bytes(g.rows, g.cols);
        lds = need > lds ? need : lds;
    }
    // more than 64 KB of dynamic LDS needs the attribute (set on every call: it is per device, and cheap)
    if (lds > 64 * 1024 && hipFuncSetAttribute((const void*)ortho_small_k<T>, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) {
        gan_set_error("orthogonalize: cannot reserve %d bytes of LDS", lds);
        return GAN_ERR_LAUNCH;
    }
    hipLaunchKernelGGL((ortho_small_k<T>), dim3((unsigned)blocks), dim3(1024), lds, st, s, h, o);
    GAN_CHECK_LAUNCH("orthogonalize(small)");
    return GAN_OK;
}

// The largest factor that a singular value can have grown to after each step, from 1: extremes of x |a + b x^2 + c x^4| on [0, r].
// growth: of the steps' factors |a + b x^2 + c x^4|, the largest product of the first ones.
bool bounded(int steps, float a, float b, float c, float& growth) {
    double r = 1.0, grown = 1.0;
    growth = 1.f;
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
        grown *= poly;
        if (grown > growth) growth = grown < 1e30 ? (float)grown : 1e30f;
    }
    return true;
}

int64_t total_bytes(const gan_matrix* mats, int count) {
    int64_t n = 0;
    bool small = true, fit = true;
    for (int k = 0; k < count; ++k) {
        const gan_matrix& g = mats[k];
        if (g.rows < 1 || g.cols < 1 || g.batch < 0 || g.rows > (1 << 20) || g.cols > (1 << 20) || g.batch >= MAXSMALL) return -1;
        if (up64(g.rows) * up64(g.cols) >= (1LL << 30) || (g.rows < g.cols ? g.rows : g.cols) > 32768) return -1;
        const Lay l = lay_of(g);
        if (g.batch && l.bytes > (1LL << 60) / g.batch) return -1;
        n += l.bytes * g.batch;
        if (n > (1LL << 60)) return -1;
        small = small && is_small(g);
        fit = fit && g.batch * blocks_of(l) < MAXBLOCKS;
    }
    return small ? 0 : fit ? n : -1;  // (small: all of them in LDS)
}

// The two launches in front of the products: momentum and norms, planes.
template <typename T>
int pack(const gan_matrix* mats, int n, char* ws, Mats& s, hipStream_t st) {
    int64_t first[2][NOPS + 1] = {};
    s.count = n;
    for (int k = 0; k < n; ++k) {
        const gan_matrix& g = mats[k];
        const Lay l = lay_of(g);
        Mat& q = s.mat[k];
        q.g = g.g;
        q.buf = g.buf;
        q.ws = ws;
        q.stride = l.bytes;
        q.x = l.x[0];
        q.rows = (int)g.rows;
        q.cols = (int)g.cols;
        ws += l.bytes * g.batch;
        const int64_t per[2] = {l.nparts, l.mp / 64 * (l.np / 64)};
        for (int j = 0; j < 2; ++j) first[j][k + 1] = first[j][k] + per[j] * g.batch;
    }
    for (int j = 0; j < 2; ++j) {
        for (int k = 0; k < n; ++k) s.first[k] = (int)first[j][k];
        const dim3 grid((unsigned)first[j][n]), block(256);
        if (j == 0) hipLaunchKernelGGL((ortho_norm_k<T>), grid, block, 0, st, s);
        else hipLaunchKernelGGL((ortho_pack_k<T>), grid, block, 0, st, s);
        GAN_CHECK_LAUNCH("orthogonalize(source)");
    }
    return GAN_OK;
}

bool all_small(const gan_matrix* mats, int count) {
    for (int k = 0; k < count; ++k)
        if (!is_small(mats[k])) return false;
    return true;
}

int run_all(const char* what, const gan_matrix* all, int count, int steps, Source source, const Rule& rule, int dtype, char* ws, int64_t bytes,
            hipStream_t st) {
    GAN_CHECK_ARG(count >= 0 && (count == 0 || all), "%s: null list", what);
    GAN_CHECK_ARG(steps >= 1 && steps <= 100, "%s: 1 to 100 steps, got %d", what, steps);
    // (SX / eps has to be a finite fp32)
    GAN_CHECK_ARG(source.eps >= 1e-30f && source.eps <= 1e30f, "%s: eps must be positive, 1e-30 to 1e30, got %g", what, (double)source.eps);
    GAN_CHECK_ARG(bounded(steps, rule.a, rule.b, rule.c, source.growth), "%s: with coefficients %g %g %g a singular value can grow beyond 3.5", what, (double)rule.a,
                  (double)rule.b, (double)rule.c);
    const int64_t need = total_bytes(all, count);
    GAN_CHECK_ARG(need >= 0, "%s: a matrix has a size that is not supported (1 to 2^20 either way, the smaller at most 32768, fewer than 2^30 elements when padded to 64s, fewer than 2^22 of them in a batch, in 2^23 blocks of 64 x 64)", what);
    GAN_CHECK_ARG(need == 0 || (ws && bytes >= need), "%s: workspace of %lld bytes wanted, %lld given", what, (long long)need,
                  (long long)(ws ? bytes : 0));
    GAN_CHECK_ARG(((uintptr_t)ws % 256) == 0, "%s: workspace must be 256-byte aligned", what);
    const bool small = all_small(all, count);
    for (int k = 0; k < count; ++k) GAN_CHECK_ARG(!all[k].batch || (all[k].g && all[k].out && (!rule.update || all[k].buf)), "%s: null pointer", what);
    Mats s = {};
    Ops o = {};
    s.from = source;
    o.rule = rule;
    gan_matrix some[NOPS];
    char* at = ws;
    for (int from = 0; from < count;) {
        int n = 0;
        int64_t used = 0, blocks = 0;
        for (; from < count && n < NOPS; ++from) {
            const gan_matrix& g = all[from];
            if (!g.batch) continue;
            const Lay l = lay_of(g);
            blocks += g.batch * (small ? 1 : blocks_of(l));
            if (n && blocks >= (small ? MAXSMALL : MAXBLOCKS)) break;  // (the next launches')
            some[n++] = g;
            if (!small) used += l.bytes * g.batch;
        }
        if (!n) break;
        if (small) {
            if (int rc = dtype == GAN_F32 ? run_small<float>(some, n, steps, source, rule, st) : run_small<bf16>(some, n, steps, source, rule, st)) return rc;
            continue;
        }
        int rc = dtype == GAN_F32 ? pack<float>(some, n, at, s, st) : pack<bf16>(some, n, at, s, st);
        if (rc) return rc;
        Walk walks[NOPS];
        int64_t tiles = 0;
        for (int k = 0; k < n; ++k) {
            walks[k] = Walk{lay_of(some[k]), false, false, steps, 1, 0, 0};
            tiles += tiles_of(walks[k].l.mp, walks[k].l.mp, true, 64) * some[k].batch;
        }
        for (int k = 0; k < n; ++k) {
            walks[k].beside = 2 * n <= NOPS && 2 * tiles <= 256;
            walks[k].pairs = two_at_a_time(walks[k].l, some[k].batch, walks[k].beside, n > 1);
        }
        for (bool more = true; more;) {
            if ((rc = products(some, walks, n, steps, o, at, dtype, st))) return rc;
            more = false;
            for (int k = 0; k < n; ++k) more |= walks[k].left > 0;
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
    return run_all("orthogonalize", mats, count, steps, Source{0.f, eps, 0, 1.f}, Rule{a, b, c, 1.f, 0.f, 0}, dtype, (char*)ws, ws_bytes, (hipStream_t)stream);
}

extern "C" int gan_muon_step(const gan_matrix* mats, int count, float lr, float momentum, int nesterov, float weight_decay, int scaling, int steps,
                             float a, float b, float c, float eps, void* ws, int64_t ws_bytes, gan_stream_t stream) {
    GAN_CHECK_ARG(lr >= 0.f && momentum >= 0.f && momentum < 1.f && weight_decay >= 0.f,
                  "muon_step: bad hyper-parameters (lr %g, momentum %g, weight_decay %g)", (double)lr, (double)momentum, (double)weight_decay);
    GAN_CHECK_ARG(scaling >= 0 && scaling <= 2, "muon_step: bad scaling %d", scaling);
    return run_all("muon_step", mats, count, steps, Source{momentum, eps, nesterov, 1.f}, Rule{a, b, c, 1.f - lr * weight_decay, lr, 1 + scaling}, GAN_F32,
                   (char*)ws, ws_bytes, (hipStream_t)stream);
}
