// muon.hip -- orthogonalisation of matrices by Newton-Schulz products, its pullback, and the Muon update that is built on it.
//
// The mathematics.  X0 = X / max(|X|_F, eps), taken with its short side first (m rows, n >= m columns), and `steps` times
//     A = X X^T,   B = b A + c A A,   X <- a X + B X          (an odd quintic in the singular values of X; nothing else of X changes).
// The pullback walks the iterates back, G = dL/dX_{k+1} -> dL/dX_k, with the symmetric S = G X^T + X G^T:
//     dL/dX_k = a G + B G + V X,   V = b S + c (S A + A S),
// and goes through the normalisation: dX = (G - X0 <X0, G>) / |X|_F   (G / eps where the norm was clamped).
// Every product is one of two forms: a symmetric result L R^T whose K axis is contiguous in both operands, of which the tiles on and above the diagonal are computed and the
// others mirrored; or (symmetric) x (m x n), whose right operand is read transposed out of LDS.  Both take a sum of two products, so S, V and the pullback's last line are one launch.
//
// Numbers.  A singular value grows by up to a per step, so what is rounded in an early step is amplified by up to a^steps (485 with the default coefficients): operands of 8 or
// 11 bits leave errors of 1e-3 .. 4e-3 relative to the result.  Every operand is therefore a PAIR of f16, x = hi + lo with 22 significant bits, and a product three
// v_mfma_f32_32x32x16_f16 (hi hi + hi lo + lo hi) with fp32 sums: 1.0 - 1.2x the error of plain fp32 products against 64 bits, at a third of the f16 rate instead of the fp32 MFMA's
// sixteenth.  The pairs are scaled by powers of two that come from bounds of the iterates' norms (ns_bounds), so that no hi overflows and the lo of a typical entry is a normal number.
// a X is added in fp32 in the epilogue: inside B (B + a I) its rounding would be the largest error of all.  Norms are sums in 64 bits.
//
// Layout.  A pair matrix is row-major in blocks of 16 columns, 64 bytes each: 16 hi, then 16 lo -- what an MFMA K-step reads of a row is contiguous.  Rows are padded to 128,
// columns of X to 128, with zeros that every step keeps (rows of B beyond m are 0), so the products need no bounds checks.  A thin matrix pays for that in memory: 1 x 2^20 fp32 (4 MB) that
// does not fit a workgroup takes 1.1 GB of workspace, 3.8 GB for its pullback (every iterate of five steps), 17 x 3 x 9000 (1.8 MB) 164 and 570 MB.
#include "md2_internal.h"
#include "muon.h"
#include <cmath>
#include <algorithm>
#include <vector>

namespace md2 {

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

namespace {

constexpr int PAD = 128;                  // rows of a pair matrix are padded to this, columns of X too
constexpr int PK_ROWS = 64, PK_COLS = 128;   // tile of the norm / pack kernels
enum { GRAM = 0, POLY = 1, SYM_S = 2, SYM_V = 3, SYMS = 4 };      // the symmetric products: A = X X^T | B = b A + c A A | S = G X^T + X G^T | V = b S + c (S A + A S)
constexpr int PART = 64 * 64 * 4;         // unit of the split products' partial sums, bytes

// where one weight (or batch of equal matrices) has its part of a product's lists
struct Use { int32_t first, red, part; };                        // first item, first reduction item, first partial sum
struct Cut { int32_t tile, chunk; };                             // a product's tile side, and at most how many K blocks an item has: the same for every weight of a call
constexpr double SX = 8192.0, SA = 2048.0, SB = 512.0;            // scales of X (norm <= 4), A (<= 16) and B (<= 60): below 2^15, and f16 ends at 65504
// what the host passes per weight, by value
struct Desc {
    const void* x; const void* d; void* y;                    // matrix | dout | result;  Muon: momentum | gradient | weight
    int64_t ws0, ws1;                                         // first matrix's buffers (bytes into the workspace), bytes per matrix
    int32_t m, n, batch, first, pk0, nn0;                     // short side, long side, matrices, index of the first, first work items
    float alpha; int32_t tall;                                // Muon: lr * shape factor | the short side is the columns
};
struct Strides { int64_t xb, xs, xl, db, ds, dl; };              // in elements: batch, along the short side, along the long side
template <int N, int KINDS> struct DescPack { Desc d[N]; Use u[N][KINDS]; };
constexpr int MUON_DESCS = 38;            // 38 * (72 + 2 * 12) bytes: a first launch's arguments stay below 4 KB

// the same per matrix, on the device
struct Mat {
    const char* x; const char* d; char* y;
    int64_t xs, xl, ds, dl, ys, yl;
    char* buf; int64_t xbytes, abytes;                        // pair buffers: nX of mp x np, then nA of mp x mp (4 bytes an entry)
    int32_t m, n, mp, np, pk0, pkn, nn0, nnn;
    float alpha;
};
// one workgroup's work; everything a product needs before its first load is in here
struct Item { char* buf; int32_t m, n, mat, ti, tj, tile, k0, k1, part, pad; };      // K blocks [k0, k1); part: where the partial sum goes, -1 = the result itself (reduction: k1 = how many)

struct Fac { float inv2; int q; };                             // a clamped matrix is carried 2^q larger (ns_pack_kernel): 2^-2q, q
struct Ws { Mat* mats; Item *sym[SYMS], *red[SYMS], *nn, *pk; Fac* fac; double* part; char* split; char* buf; };      // part: [2][pk items] sums of squares of x, of dout, and [nn items] of X0 G

__host__ __device__ inline int cdiv(int a, int b) { return (a + b - 1) / b; }
__host__ __device__ inline int kblocks(int kind, int m, int n) { return (kind >= SYM_S ? 2 : 1) * cdiv(kind == GRAM || kind == SYM_S ? n : m, 16); }

struct Cuts { Cut sym[SYMS]; int32_t nn_tile, fuse; };           // fuse: every short side is at most 64 (sym_whole): 64-tiles throughout, GRAM and SYM_S do POLY's and SYM_V's work
// Workgroup b runs on XCD b % 8, each with an L2 of its own.  Of `groups` groups of `size` items, the items of one share an operand: eight groups at a time are dealt to the XCDs, a group
// to one.  -> the place of item `i` of group `g` (the last groups, fewer than eight, are dealt among themselves)
__device__ inline int dealt(int g, int i, int groups, int size) {
    const int full = groups / 8 * 8, r = groups - full;
    return g < full ? g / 8 * 8 * size + i * 8 + g % 8 : full * size + i * r + (g - full);
}
// matrix b of a weight (or of a batch with strides of its own, N = 1)
template <int N> __device__ inline Mat make_mat(const Desc& D, const Strides& st, const Cuts& cuts, int dt_bytes, char* base, int b) {
    const int mp = cdiv(D.m, PAD) * PAD, np = cdiv(D.n, PAD) * PAD, npk = mp / PK_ROWS * (np / PK_COLS), nnn = cdiv(D.m, cuts.nn_tile) * cdiv(D.n, cuts.nn_tile);
    const int64_t ss = D.tall ? 1 : D.n, sl = D.tall ? D.m : 1;      // a contiguous matrix's strides
    Mat M;
    M.x = (const char*)D.x + (N == 1 ? st.xb * b * dt_bytes : 0); M.d = (const char*)D.d + (N == 1 ? st.db * b * dt_bytes : 0); M.y = (char*)D.y + (int64_t)D.m * D.n * b * dt_bytes;
    M.xs = N == 1 ? st.xs : ss; M.xl = N == 1 ? st.xl : sl; M.ds = N == 1 ? st.ds : ss; M.dl = N == 1 ? st.dl : sl; M.ys = ss; M.yl = sl;
    M.buf = base + D.ws0 + D.ws1 * b; M.m = D.m; M.n = D.n; M.mp = mp; M.np = np;
    M.xbytes = (int64_t)mp * np * 4; M.abytes = (int64_t)mp * mp * 4;
    M.pk0 = D.pk0 + npk * b; M.pkn = npk; M.nn0 = D.nn0 + nnn * b; M.nnn = nnn; M.alpha = D.alpha;
    return M;
}
// the tables and work lists of a weight's matrices first, first + by, ...
template <int N, int KINDS> __device__ inline void set_up(const Desc& D, const Use* use, const Strides& st, const Cuts& cuts, int dt_bytes, const Ws& ws, int first, int by) {
    const int mp = cdiv(D.m, PAD) * PAD, np = cdiv(D.n, PAD) * PAD, npk = mp / PK_ROWS * (np / PK_COLS), pr = mp / PK_ROWS, nr = cdiv(D.m, cuts.nn_tile), nnn = nr * cdiv(D.n, cuts.nn_tile);
    for (int b = first; b < D.batch; b += by) {
        const int id = D.first + b; char* buf = ws.buf + D.ws0 + D.ws1 * b;
        if (threadIdx.x == 0) ws.mats[id] = make_mat<N>(D, st, cuts, dt_bytes, ws.buf, b);
#pragma unroll
        for (int kind = 0; kind < KINDS; ++kind) {
            const Use& u = use[kind]; const Cut cut = cuts.sym[kind];
            const int mt = cdiv(D.m, cut.tile), tri = mt * (mt + 1) / 2, kb = kblocks(kind, D.m, D.n), per = cut.tile * cut.tile * 4 / PART, chunk = cdiv(kb, cdiv(kb, cut.chunk)), split = cdiv(kb, chunk);
            for (int q = threadIdx.x; q < mt * mt; q += 256) {
                const int i = q / mt, j = q % mt;
                if (j < i) continue;
                const int own = i * mt - i * (i - 1) / 2 + (j - i), e = tri * b + own, part = u.part + e * split * per;
                for (int k = 0; k < split; ++k)      // (the tiles of one piece of the K axis read the same columns)
                    ws.sym[kind][u.first + tri * b * split + dealt(k, own, split, tri)] = Item{buf, D.m, D.n, id, i, j, cut.tile, k * chunk, min(kb, (k + 1) * chunk), split > 1 ? part + k * per : -1, 0};
                if (split > 1) ws.red[kind][u.red + e] = Item{buf, D.m, D.n, id, i, j, cut.tile, 0, split, part, 0};
            }
        }
        for (int q = threadIdx.x; q < nnn; q += 256) ws.nn[D.nn0 + nnn * b + dealt(q / nr, q % nr, nnn / nr, nr)] = Item{buf, D.m, D.n, id, q % nr, q / nr, cuts.nn_tile, 0, 0, 0, 0};
        for (int q = threadIdx.x; q < npk; q += 256) ws.pk[D.pk0 + npk * b + q] = Item{buf, D.m, D.n, id, q % pr, q / pr, 0, 0, 0, 0, 0};
    }
}

// ---- elements ---------------------------------------------------------------------------------------------------------
template <int DT> __device__ inline float ld_el(const char* p, int64_t i) {
    if constexpr (DT == NS_F32) return reinterpret_cast<const float*>(p)[i];
    else if constexpr (DT == NS_F16) return (float)reinterpret_cast<const _Float16*>(p)[i];
    else return __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(p)[i] << 16);
}
template <int DT> __device__ inline void st_el(char* p, int64_t i, float v) {
    if constexpr (DT == NS_F32) reinterpret_cast<float*>(p)[i] = v;
    else if constexpr (DT == NS_F16) reinterpret_cast<_Float16*>(p)[i] = (_Float16)v;
    else { const uint32_t u = __float_as_uint(v); reinterpret_cast<uint16_t*>(p)[i] = v != v ? (uint16_t)((u >> 16) | 0x40) : (uint16_t)((u + 0x7fff + ((u >> 16) & 1)) >> 16); }
}
// (v is pinned: left to itself the compiler folds the multiplication that made it into the conversion to hi, but not into the difference, and where v lies next to a tie of f16 the
// two then disagree about hi by one of its steps)
__device__ inline void split4(const float v[4], f16x4& hi, f16x4& lo) {
#pragma unroll
    for (int e = 0; e < 4; ++e) { float x = v[e]; asm("" : "+v"(x)); hi[e] = (_Float16)x; lo[e] = (_Float16)(x - (float)hi[e]); }
}
constexpr int LO = 32;                    // bytes from a hi to its lo
__device__ inline int64_t pair_off(int64_t row_bytes, int i, int j) { return i * row_bytes + (j >> 4) * 64 + (j & 15) * 2; }      // bytes of hi(i, j)

// sum over the block in a fixed order (256 threads); every thread gets it
__device__ inline double block_sum(double v, double* red) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

struct MuonArgs { float beta, rest, gscale; int nesterov; };      // rest = 1 - beta, rounded once: 1.f - beta loses it as beta nears 1
enum { SRC_X = 0, SRC_DOUT = 1, SRC_MUON = 2 };

// four neighbouring elements, aligned to their size together
template <int DT> __device__ inline f32x4 ld_el4(const char* p, int64_t i) {
    if constexpr (DT == NS_F32) return *reinterpret_cast<const f32x4*>(p + i * 4);
    else {
        const s16x4 q = *reinterpret_cast<const s16x4*>(p + i * 2); f32x4 r;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = DT == NS_F16 ? (float)__builtin_bit_cast(_Float16, (short)q[e]) : __uint_as_float((uint32_t)(uint16_t)q[e] << 16);
        return r;
    }
}
__device__ inline float momentum_step(float m, float g, const MuonArgs& mu) { return mu.beta * m + mu.rest * (mu.gscale * g); }
__device__ inline float muon_u(float m, float g, const MuonArgs& mu) { return mu.nesterov ? mu.beta * m + mu.rest * (mu.gscale * g) : m; }
// One 64 x 128 tile of the source, 8 values of each of the thread's four columns: v[p][e] = element (p * 8 + t / 32, (t % 32) * 4 + e).
// Rows whose long side is contiguous and aligned are read as vectors; any other source element by element along its contiguous side (neighbouring lanes, neighbouring addresses) and
// through LDS.  All of a thread's loads are issued before the first is used: what lies outside reads the first row or element instead and is dropped (behind a branch each 16-bit load
// waited for its conversion: 10 - 12 us a launch against 6).  UPDATE: the momentum moves on and is written back.
template <int DT, int SRC, bool UPDATE> __device__ inline void load_tile(const Mat& M, const Item& it, const MuonArgs& mu, float v[8][4], float* lds) {
    const int t = threadIdx.x, i0 = it.ti * PK_ROWS, j0 = it.tj * PK_COLS; constexpr int EL = DT == NS_F32 ? 4 : 2;
    const char* src = SRC == SRC_DOUT ? M.d : M.x; const int64_t ss = SRC == SRC_DOUT ? M.ds : M.xs, sl = SRC == SRC_DOUT ? M.dl : M.xl;
    float* mom = reinterpret_cast<float*>(const_cast<char*>(M.x));
    const uintptr_t align = reinterpret_cast<uintptr_t>(src) | (SRC == SRC_MUON ? reinterpret_cast<uintptr_t>(M.d) : 0);
    if (sl == 1 && align % (4 * EL) == 0 && ss % 4 == 0 && j0 + PK_COLS <= M.n) {
        f32x4 x[8], g[8]; const int j = j0 + (t & 31) * 4;
#pragma unroll
        for (int p = 0; p < 8; ++p) {
            const int i = i0 + p * 8 + (t >> 5); const int64_t o = (i < M.m ? i * ss : 0) + j;
            x[p] = ld_el4<DT>(src, o);
            if constexpr (SRC == SRC_MUON) g[p] = *reinterpret_cast<const f32x4*>(M.d + o * 4);
        }
#pragma unroll
        for (int p = 0; p < 8; ++p) if (i0 + p * 8 + (t >> 5) >= M.m) { x[p] = f32x4{0, 0, 0, 0}; if constexpr (SRC == SRC_MUON) g[p] = f32x4{0, 0, 0, 0}; }
#pragma unroll
        for (int p = 0; p < 8; ++p) {
            const int i = i0 + p * 8 + (t >> 5);
            if constexpr (SRC == SRC_MUON && UPDATE) {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[p][e] = momentum_step(x[p][e], g[p][e], mu);
                if (i < M.m) *reinterpret_cast<f32x4*>(mom + i * ss + j) = x[p];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) v[p][e] = SRC == SRC_MUON ? muon_u(x[p][e], g[p][e], mu) : x[p][e];
        }
        return;
    }
    const bool turn = ss == 1 && sl != 1;
#pragma unroll (SRC == SRC_MUON ? 1 : 2)
    for (int h = 0; h < 2; ++h) {
        float x[16], g[16];
        auto at = [&](int q, int& i, int& j) { const int id = h * 4096 + q * 256 + t; i = turn ? id & 63 : id >> 7; j = turn ? id >> 6 : id & 127; };
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            int i, j; at(q, i, j); const bool in = i0 + i < M.m && j0 + j < M.n; const int64_t o = in ? (i0 + i) * ss + (j0 + j) * sl : 0;
            x[q] = ld_el<DT>(src, o);
            if constexpr (SRC == SRC_MUON) g[q] = reinterpret_cast<const float*>(M.d)[o];
            x[q] = in ? x[q] : 0.f;
            if constexpr (SRC == SRC_MUON) g[q] = in ? g[q] : 0.f;
        }
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            int i, j; at(q, i, j);
            if constexpr (SRC == SRC_MUON && UPDATE) {
                x[q] = momentum_step(x[q], g[q], mu);
                if (i0 + i < M.m && j0 + j < M.n) mom[(i0 + i) * ss + (j0 + j) * sl] = x[q];
            }
            lds[i * (PK_COLS + 1) + j] = SRC == SRC_MUON ? muon_u(x[q], g[q], mu) : x[q];
        }
    }
    __syncthreads();
#pragma unroll
    for (int p = 0; p < 8; ++p)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[p][e] = lds[(p * 8 + (t >> 5)) * (PK_COLS + 1) + (t & 31) * 4 + e];
}

// A call's first launch: the tables and work lists of the later ones (the first `tables` workgroups), and the sum of squares of every tile (Muon: after moving the momentum on; the
// pullback's second half of the grid: of dout's), which work their tiles out themselves.  As launches of their own the tables cost 5 - 13 us, which now pass beside the sums.
template <int DT, int SRC, int N, int KINDS> __global__ __launch_bounds__(256) void ns_start_kernel(DescPack<N, KINDS> dp, int weights, int tables, int tiles, Strides st, Cuts cuts, Ws ws, MuonArgs mu) {
    __shared__ float lds[PK_ROWS * (PK_COLS + 1)]; __shared__ double red[4]; constexpr int BYTES = DT == NS_F32 ? 4 : 2;
    if (blockIdx.x < tables) {
        const int w = N == 1 ? 0 : blockIdx.x;
        if (blockIdx.y == 0) set_up<N, KINDS>(dp.d[w], dp.u[w], st, cuts, BYTES, ws, N == 1 ? blockIdx.x : 0, N == 1 ? tables : 1);
        return;
    }
    const int id = dp.d[0].pk0 + blockIdx.x - tables; int w = 0;
    if constexpr (N > 1) for (int hi = weights - 1; w < hi;) { const int q = (w + hi + 1) / 2; if (dp.d[q].pk0 <= id) w = q; else hi = q - 1; }
    const Desc& D = dp.d[w]; const int pr = cdiv(D.m, PAD) * PAD / PK_ROWS, npk = pr * cdiv(D.n, PAD) * (PAD / PK_COLS), b = (id - D.pk0) / npk, q = (id - D.pk0) % npk;
    const Mat M = make_mat<N>(D, st, cuts, BYTES, ws.buf, b); Item it{}; it.ti = q % pr; it.tj = q / pr;
    float v[8][4];
    if (SRC == SRC_X && blockIdx.y) load_tile<DT, SRC_DOUT, false>(M, it, mu, v, lds); else load_tile<DT, SRC, true>(M, it, mu, v, lds);
    double s = 0;
#pragma unroll
    for (int p = 0; p < 8; ++p)
#pragma unroll
        for (int e = 0; e < 4; ++e) s += (double)v[p][e] * (double)v[p][e];
    s = block_sum(s, red);
    if (threadIdx.x == 0) ws.part[blockIdx.y * tiles + id] = s;
}
// |.|_F of a matrix from its tiles' sums, in a fixed order
__device__ inline double norm_of(const Mat& M, const double* part, double* red) {
    double s = 0;
    for (int q = threadIdx.x; q < M.pkn; q += 256) s += part[M.pk0 + q];
    return sqrt(block_sum(s, red));
}
// scale * source / max(norm, eps) as pairs; the pullback's second half of the grid: d_scale * dout / |dout| into d_slot.
// Where the norm r = |X| / eps is clamped, X0 may be too small for f16: it is carried 2^q larger, 2^q r grow <= 4 (grow: by how much all steps can grow a singular value; the pullback: Plan::carry), so A, B, S and V
// are 2^2q, 2^2q, 2^q and 2^q larger, and what has one factor of A too many (A A, S A, B X, V X) is multiplied by 2^-2q.  q = 0 for every other matrix.
template <int DT, int SRC> __global__ __launch_bounds__(256) void ns_pack_kernel(Ws ws, MuonArgs mu, double scale, double eps, double grow, int d_slot, double d_scale) {
    __shared__ float lds[PK_ROWS * (PK_COLS + 1)]; __shared__ double red[4];
    const Item it = ws.pk[blockIdx.x]; const Mat M = ws.mats[it.mat]; const bool dout = SRC == SRC_X && blockIdx.y;
    float v[8][4];                                               // (before the norm: its sums wait for memory too)
    if (dout) load_tile<DT, SRC_DOUT, false>(M, it, mu, v, lds); else load_tile<DT, SRC, false>(M, it, mu, v, lds);
    const double norm = norm_of(M, ws.part + (dout ? gridDim.x : 0), red);
    if (dout) { scale = d_scale; eps = 0; }
    else {
        int q = 0;
        if (norm <= eps && norm > 0) { const double room = 4.0 * eps / (norm * grow); if (room >= 2.0) q = ilogb(room); }
        if (it.ti == 0 && it.tj == 0 && threadIdx.x == 0) ws.fac[it.mat] = Fac{(float)ldexp(1.0, -2 * q), q};
        scale = ldexp(scale, q);
    }
    const double fd = norm <= eps ? (norm > 0 ? scale / eps : 0.0) : scale / norm;     // (a NaN norm stays one; zeros stay zeros, however small eps is)
    int fe; const float f = (float)frexp(fd, &fe);               // mantissa and exponent apart: 1 / norm may lie outside fp32's range where the product does not
    char* out = M.buf + (dout ? d_slot : 0) * M.xbytes; const int64_t rb = (int64_t)M.np * 4;
#pragma unroll
    for (int p = 0; p < 8; ++p) {
        float w[4]; f16x4 hi, lo;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = ldexpf(v[p][e], fe) * f;
        split4(w, hi, lo);
        char* o = out + pair_off(rb, it.ti * PK_ROWS + p * 8 + (threadIdx.x >> 5), it.tj * PK_COLS + (threadIdx.x & 31) * 4);
        *reinterpret_cast<f16x4*>(o) = hi; *reinterpret_cast<f16x4*>(o + LO) = lo;
    }
}

// ---- products -------------------------------------------------------------------------------------------------------------
struct Slot { int x, a; };                                                      // buffer = x * xbytes + a * abytes behind the matrix's first
__device__ inline char* slot(const Mat& M, Slot s) { return M.buf + s.x * M.xbytes + s.a * M.abytes; }
struct Dims { int64_t xrb, arb, xbytes, abytes; };                              // row bytes and buffer bytes of X's and of A's kind
__device__ inline Dims dims(const Item& it) {
    const int mp = cdiv(it.m, PAD) * PAD, np = cdiv(it.n, PAD) * PAD;
    return Dims{(int64_t)np * 4, (int64_t)mp * 4, (int64_t)mp * np * 4, (int64_t)mp * mp * 4};
}
__device__ inline char* slot(const Item& it, const Dims& d, Slot s) { return it.buf + s.x * d.xbytes + s.a * d.abytes; }

typedef __attribute__((address_space(3))) void* lds_t;
// LDS of a product: RING stages of 16 K of both operands.  128-tiles: shared by the workgroup, 16 KB each, so that two workgroups share a CU; 64-tiles: each wave's own, 8 KB each
template <int T> struct Ring { static constexpr int N = T == 128 ? 5 : 4, STAGE = T == 128 ? 16384 : 8192, THREADS = T == 128 ? 256 : 64, LOADS = STAGE / THREADS / 32, BYTES = T == 128 ? N * STAGE : 4 * N * STAGE; };      // LOADS: a wave's instructions per stage and operand

// Direct loads (global memory -> LDS, 16 bytes a lane; a wave writes 1 KB in lane order, so the bank swizzle is in which chunk a lane FETCHES).  Written as assembly because the compiler
// lets a transposed LDS read wait for every direct load in flight that it knows of; it has no register result, and the product counts and waits itself.
__device__ inline void direct_load(unsigned lds, const char* base, unsigned off) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" :: "s"(lds), "v"(off), "s"(base) : "memory");
}
// Rows: T x 16 columns of a pair matrix; row r's four 16-byte chunks (hi k 0..7, 8..15, lo 0..7, 8..15) are stored at chunk ^ row_swizzle(r), which spreads neighbouring rows' reads of one
// chunk over the 64 banks (four rows wide).
__device__ inline int row_swizzle(int r) { return ((r >> 2) & 1) | ((((r >> 1) ^ (r >> 3)) & 1) << 1); }
// Columns: 16 rows (the K axis) x T columns; a row's 32-byte units are stored at unit ^ col_swizzle(k), so that the four rows and two units of 32 lanes' transposed read meet eight
// different places of the 64 banks
__device__ inline int col_swizzle(int k) { return (k & 1) | (((k >> 1) & 1) << 2) | (((k >> 3) & 1) << 1); }
// a lane's bytes behind the stage's first, per instruction
template <int T, bool COLS> __device__ inline void lane_offsets(unsigned off[Ring<T>::LOADS], int64_t rb, int tid) {
#pragma unroll
    for (int q = 0; q < Ring<T>::LOADS; ++q) {
        const int id = q * Ring<T>::THREADS + tid;
        if constexpr (COLS) { constexpr int CH = T / 4; const int k = id / CH; off[q] = (unsigned)(k * rb) + ((id % CH) ^ (col_swizzle(k) << 1)) * 16; }
        else { const int r = id >> 2; off[q] = (unsigned)(r * rb) + ((id & 3) ^ row_swizzle(r)) * 16; }
    }
}
__device__ inline f16x8 frag_rows(const char* lds, int r, int c) { return *reinterpret_cast<const f16x8*>(lds + r * 64 + ((c ^ row_swizzle(r)) << 4)); }
// The MFMA operands of 64 columns from c0 (two of 32) and 16 rows (lane: column lane % 32, rows (lane / 32) * 8 .. + 8), hi and lo.
// ds_read_b64_tr_b16: within 16 lanes, lane s gives the address of 4 columns of row s / 4 and receives the four rows of column s; two reads, four rows apart, make an operand.
// 32 columns on and lo each flip one bit of the swizzled unit (128 and 32 bytes).
template <int T> __device__ inline unsigned cols_at(int c0) {
    const int l = threadIdx.x & 63, s = l & 15, g = l >> 4, k = (g >> 1) * 8 + (s >> 2), col = c0 + (g & 1) * 16 + (s & 3) * 4;
    return k * (T * 4) + ((((col >> 4) * 2) ^ col_swizzle(k)) << 5) + (col & 15) * 2;
}
template <int T> __device__ inline f16x8 frag_cols(unsigned at) {
    typedef __attribute__((address_space(3))) s16x4* p4;
    const s16x4 u = __builtin_amdgcn_ds_read_tr16_b64_v4i16((p4)(uintptr_t)at), v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((p4)(uintptr_t)(at + 4 * T * 4));
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    return __builtin_bit_cast(f16x8, (s16x8)__builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7));
}
struct Frags { f16x8 ah[2], al[2], bh[2], bl[2]; };              // [32 columns of the wave's 64]

// One operand pair of a product: a's and b's first bytes and what a K block of 16 advances them by
struct Seg { const char *a, *b; int64_t arb, brb, ak, bk; };
// sum over the K blocks [k0, k1) of a b^T (NN: a's K axis runs along its rows).  The blocks of the second segment begin at `kb`; c is multiplied by `mid` there.
// T = 128: four waves of 64 x 64, operands staged for all of them.  T = 64: every wave has the whole tile and each fourth K block, LDS of its own and no barrier; the four sums meet in
// the epilogue.
// Per step of 16 K (384 cycles of MFMAs a wave): wait for the next stage's loads, counted -- the younger stages' stay in flight, RING - 1 steps ahead, a way from memory -- and for this
// step's operands, which were read during the last step's MFMAs; barrier; then a third of the MFMAs, the next operands' reads, a third, the loads into the stage just freed, a third.
// The statements with a memory clobber keep LDS reads where they are (its address went into the direct loads); the operands go through the one that ends their reads.
template <int T, bool NN> __device__ inline void product(char* lds, const Seg seg[2], int kb, int k0, int k1, float mid, f32x16 c[2][2]) {
    using R = Ring<T>;
    const int t = threadIdx.x, lane = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6), lr = lane & 31, lk = lane >> 5;
    constexpr int step = T == 128 ? 1 : 4, HALF = R::STAGE / 2; const int wa = T == 128 ? (wv >> 1) * 64 : 0, wb = T == 128 ? (wv & 1) * 64 : 0;
    char* ring = lds + (T == 128 ? 0 : wv * R::N * R::STAGE); const unsigned ring_at = (unsigned)(uintptr_t)(lds_t)ring, mine = ring_at + (T == 128 ? wv * 1024 : 0), cols = NN ? cols_at<T>(wa) + ring_at : 0;
    unsigned oa[R::LOADS], ob[R::LOADS];
    lane_offsets<T, NN>(oa, seg[0].arb, T == 128 ? t : lane); lane_offsets<T, false>(ob, seg[0].brb, T == 128 ? t : lane);
    auto issue = [&](int k, int at) {
        const bool s2 = k >= kb; const int kk = s2 ? k - kb : k;
        const char *pa = (s2 ? seg[1].a : seg[0].a) + kk * seg[0].ak, *pb = (s2 ? seg[1].b : seg[0].b) + kk * seg[0].bk;
#pragma unroll
        for (int q = 0; q < R::LOADS; ++q) { direct_load(mine + at + q * R::THREADS * 16, pa, oa[q]); direct_load(mine + at + HALF + q * R::THREADS * 16, pb, ob[q]); }
    };
    auto read = [&](Frags& f, int at) {
        const char *la = ring + at, *lb = la + HALF;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            if constexpr (NN) { const unsigned u = (cols ^ (q * 128)) + at; f.ah[q] = frag_cols<T>(u); f.al[q] = frag_cols<T>(u ^ 32); }
            else { f.ah[q] = frag_rows(la, wa + q * 32 + lr, lk); f.al[q] = frag_rows(la, wa + q * 32 + lr, lk + 2); }
            f.bh[q] = frag_rows(lb, wb + q * 32 + lr, lk); f.bl[q] = frag_rows(lb, wb + q * 32 + lr, lk + 2);
        }
    };
    const int first = k0 + (T == 128 ? 0 : wv); bool second = first >= kb;
    if (first < k1) {
#pragma unroll
        for (int i = 0; i < R::N; ++i) if (first + i * step < k1) issue(first + i * step, i * R::STAGE);
        if (first + (R::N - 1) * step < k1) asm volatile("s_waitcnt vmcnt(%0)" :: "n"((R::N - 1) * 2 * R::LOADS) : "memory"); else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if constexpr (T == 128) asm volatile("s_barrier" ::: "memory");
        Frags f0, f1; int at = 0;
        read(f0, 0);
        auto turn = [&](Frags& f, Frags& next, int k) {
            const int on = at == (R::N - 1) * R::STAGE ? 0 : at + R::STAGE; const bool more = k + step < k1, load = k + R::N * step < k1;
            if (k + (R::N - 1) * step < k1) asm volatile("s_waitcnt vmcnt(%0)" :: "n"((R::N - 2) * 2 * R::LOADS) : "memory"); else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(f.ah[0]), "+v"(f.al[0]), "+v"(f.bh[0]), "+v"(f.bl[0]), "+v"(f.ah[1]), "+v"(f.al[1]), "+v"(f.bh[1]), "+v"(f.bl[1]) :: "memory");
            if constexpr (T == 128) asm volatile("s_barrier" ::: "memory");
            if (!second && k >= kb) {                            // the second product's scale is another power of two
                second = true;
#pragma unroll
                for (int p = 0; p < 2; ++p)
#pragma unroll
                    for (int q = 0; q < 2; ++q) c[p][q] *= mid;
            }
            // c += (ah + al) (bh + bl) without al bl: small terms first, the four accumulators in turn (an accumulator's next product waits for its last)
#pragma unroll
            for (int p = 0; p < 2; ++p)
#pragma unroll
                for (int q = 0; q < 2; ++q) c[p][q] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.al[p], f.bh[q], c[p][q], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
            if (more) read(next, on);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int p = 0; p < 2; ++p)
#pragma unroll
                for (int q = 0; q < 2; ++q) c[p][q] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.ah[p], f.bl[q], c[p][q], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
            if (load) issue(k + R::N * step, at);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int p = 0; p < 2; ++p)
#pragma unroll
                for (int q = 0; q < 2; ++q) c[p][q] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.ah[p], f.bh[q], c[p][q], 0, 0, 0);
            at = on;
        };
        for (int k = first; k < k1; k += 2 * step) {
            turn(f0, f1, k);
            if (k + step < k1) turn(f1, f0, k + step);
        }
    }
    if (!second && kb < k1)                                      // (this wave's share ended before the second product)
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int q = 0; q < 2; ++q) c[p][q] *= mid;
}

// The tile in LDS as fp32, rows = b's axis, columns = a's: 16-byte units at unit ^ row, so that writes along the lanes' rows and reads along a row both meet every bank
template <int T> __device__ inline int tile_at(int r, int c) { return r * T + ((((c >> 2) ^ r) & (T / 4 - 1)) << 2) + (c & 3); }
template <int T> __device__ inline void tile_store(float* tile, const f32x16 c[2][2]) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, lr = lane & 31, lk = lane >> 5, wa = T == 128 ? (wv >> 1) * 64 : 0, wb = T == 128 ? (wv & 1) * 64 : 0;
    float* l = tile + (T == 128 ? 0 : wv * 64 * 64);
    __syncthreads();                                             // the staged operands have been read by every wave
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                f32x4 w;
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = c[p][q][g * 4 + e];
                *reinterpret_cast<f32x4*>(l + tile_at<T>(wb + q * 32 + lr, wa + p * 32 + g * 8 + lk * 4)) = w;
            }
    __syncthreads();
}
// eight neighbouring columns of a row; 64-tiles: of the four waves' sums
template <int T> __device__ inline void tile_row8(const float* tile, int planes, int r, int c, float v[8]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        f32x4 w = *reinterpret_cast<const f32x4*>(tile + tile_at<T>(r, c + h * 4));
        if (T == 64 && planes == 4) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(tile + 4096 + tile_at<T>(r, c + h * 4)), y = *reinterpret_cast<const f32x4*>(tile + 8192 + tile_at<T>(r, c + h * 4)),
                        z = *reinterpret_cast<const f32x4*>(tile + 12288 + tile_at<T>(r, c + h * 4));
            w = (w + x) + (y + z);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) v[h * 4 + e] = w[e];
    }
}
template <int T> __device__ inline float tile_el(const float* tile, int planes, int r, int c) {
    const int o = tile_at<T>(r, c);
    return T == 64 && planes == 4 ? (tile[o] + tile[4096 + o]) + (tile[8192 + o] + tile[12288 + o]) : tile[o];
}
__device__ inline void store_pair8(char* p, const float v[8]) {
    f16x4 h[2], l[2]; split4(v, h[0], l[0]); split4(v + 4, h[1], l[1]);
    *reinterpret_cast<f16x8*>(p) = __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7); *reinterpret_cast<f16x8*>(p + LO) = __builtin_shufflevector(l[0], l[1], 0, 1, 2, 3, 4, 5, 6, 7);
}

__device__ inline void unpack4(const f16x4 h, const f16x4 l, float v[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (float)h[e] + (float)l[e];
}
// four neighbouring columns (j a multiple of 4) of a swizzled LDS row
__device__ inline char* small_at(char* rows, int stride, int i, int j, int lo) { return rows + i * stride + (((j >> 4) ^ (i & 3)) << 6) + (((((j & 15) >> 3) + lo * 2) ^ row_swizzle(i)) << 4) + (j & 4) * 2; }
__device__ inline f16x8 small_row(const char* rows, int stride, int i, int block, int chunk) { return *reinterpret_cast<const f16x8*>(rows + i * stride + ((block ^ (i & 3)) << 6) + ((chunk ^ row_swizzle(i)) << 4)); }

struct SymArgs { Slot l[2], r[2], e, out; int kind, nseg, have_e; float acc, ecoef; Slot with, then; int fuse; float acc2, ecoef2; };      // out = acc * (sum of l r^T) + ecoef * e, in the buffers' own scales (with e: a factor A too many)
__device__ inline void unpack8(const f16x8 h, const f16x8 l, float v[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)h[e] + (float)l[e];
}
// R rows (tj's, from r0) of a tile with T columns (ti's) to their place and, off the diagonal, to their mirror image's; what is read of e is read before anything is written
template <int T, int R> __device__ inline void sym_finish(const Item& it, const SymArgs& a, const Fac* facs, const float* tile, int planes, int r0) {
    const int t = threadIdx.x; const Dims d = dims(it);
    char* out = slot(it, d, a.out); const char* E = slot(it, d, a.e); const float facc = a.have_e ? a.acc * facs[it.mat].inv2 : a.acc;
    constexpr int N = R * T / 8 / 256;                           // groups of 8 values a thread
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        if (side && it.ti == it.tj) break;
        f16x8 eh[N], el[N]; int64_t off[N];
#pragma unroll
        for (int z = 0; z < N; ++z) {
            const int id = z * 256 + t, r = side ? id / (R / 8) : id / (T / 8), c = side ? id % (R / 8) * 8 : id % (T / 8) * 8;
            off[z] = pair_off(d.arb, side ? it.ti * T + r : it.tj * T + r0 + r, side ? it.tj * T + r0 + c : it.ti * T + c);
            if (a.have_e) { eh[z] = *reinterpret_cast<const f16x8*>(E + off[z]); el[z] = *reinterpret_cast<const f16x8*>(E + off[z] + LO); }
        }
#pragma unroll
        for (int z = 0; z < N; ++z) {
            const int id = z * 256 + t, r = side ? id / (R / 8) : id / (T / 8), c = side ? id % (R / 8) * 8 : id % (T / 8) * 8; float v[8];
            if (side == 0) tile_row8<T>(tile, planes, r, c, v);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = tile_el<T>(tile, planes, c + e, r);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= facc;
            if (a.have_e) {
                float x[8]; unpack8(eh[z], el[z], x);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] += a.ecoef * x[e];
            }
            store_pair8(out + off[z], v);
        }
    }
}
// Short sides of at most 64: the workgroup that has all of A goes on to B = b A + c A A (and from S to V = b S + c (S A + A S), `with` being A), which saves a launch.  lds: 32 KB
__device__ inline void sym_whole(char* lds, const Item& it, const SymArgs& a, const Fac* facs, const float* tile, int planes) {
    const int t = threadIdx.x, lane = t & 63, lr = lane & 31, lk = lane >> 5, i0 = (t >> 7) * 32, j0 = ((t >> 6) & 1) * 32; const Dims d = dims(it);
    char *first = lds, *second = a.kind == SYM_S ? lds + 16384 : first, *out = slot(it, d, a.out), *then = slot(it, d, a.then); const char* with = slot(it, d, a.with); const float inv2 = facs[it.mat].inv2;
#pragma unroll
    for (int z = 0; z < 2; ++z) {
        const int r = z * 32 + t / 8, c = t % 8 * 8; const int64_t o = pair_off(d.arb, r, c); float v[8];
        if (a.kind == SYM_S) { *reinterpret_cast<f16x8*>(small_at(second, 256, r, c, 0)) = *reinterpret_cast<const f16x8*>(with + o); *reinterpret_cast<f16x8*>(small_at(second, 256, r, c, 1)) = *reinterpret_cast<const f16x8*>(with + o + LO); }
        tile_row8<64>(tile, planes, r, c, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= a.acc;
        f16x4 h[2], l[2]; split4(v, h[0], l[0]); split4(v + 4, h[1], l[1]);
        const f16x8 hi = __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7), lo = __builtin_shufflevector(l[0], l[1], 0, 1, 2, 3, 4, 5, 6, 7);
        *reinterpret_cast<f16x8*>(small_at(first, 256, r, c, 0)) = hi; *reinterpret_cast<f16x8*>(small_at(first, 256, r, c, 1)) = lo;
        if (a.kind == GRAM) { *reinterpret_cast<f16x8*>(out + o) = hi; *reinterpret_cast<f16x8*>(out + o + LO) = lo; }      // (the pullback reads A again; S goes no further)
    }
    __syncthreads();
    f32x16 c[3] = {};
    auto add = [&](const char* L, const char* R) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const f16x8 ah = small_row(L, 256, i0 + lr, k, lk), al = small_row(L, 256, i0 + lr, k, lk + 2), bh = small_row(R, 256, j0 + lr, k, lk), bl = small_row(R, 256, j0 + lr, k, lk + 2);
            c[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bh, c[0], 0, 0, 0); c[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al, bh, c[1], 0, 0, 0); c[2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bl, c[2], 0, 0, 0);
        }
    };
    add(first, second);
    if (a.kind == SYM_S) add(second, first);
    c[0] += c[1] + c[2];
#pragma unroll
    for (int g = 0; g < 4; ++g) {                                // lane: row j0 + lr, registers: four neighbouring columns (the result is symmetric)
        const int i = i0 + g * 8 + lk * 4, j = j0 + lr; const int64_t o = pair_off(d.arb, j, i); float x[4], v[4]; f16x4 hi, lo;
        unpack4(*reinterpret_cast<const f16x4*>(small_at(first, 256, j, i, 0)), *reinterpret_cast<const f16x4*>(small_at(first, 256, j, i, 1)), x);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = a.acc2 * inv2 * c[0][g * 4 + e] + a.ecoef2 * x[e];
        split4(v, hi, lo);
        *reinterpret_cast<f16x4*>(then + o) = hi; *reinterpret_cast<f16x4*>(then + o + LO) = lo;
    }
}
template <int T> __device__ inline void sym_tile(char* lds, const Item& it, const Ws& ws, const SymArgs& a) {
    const Dims d = dims(it); const bool kn = a.kind == GRAM || a.kind == SYM_S; const int64_t rb = kn ? d.xrb : d.arb;
    Seg seg[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) seg[s] = Seg{slot(it, d, a.l[s]) + (int64_t)it.ti * T * rb, slot(it, d, a.r[s]) + (int64_t)it.tj * T * rb, rb, rb, 64, 64};
    f32x16 c[2][2] = {};
    product<T, false>(lds, seg, a.nseg == 2 ? cdiv(kn ? it.n : it.m, 16) : 1 << 30, it.k0, it.k1, 1.f, c);
    float* tile = reinterpret_cast<float*>(lds); tile_store<T>(tile, c);
    if (T == 64 && it.part < 0 && a.fuse) sym_whole(lds + 65536, it, a, ws.fac, tile, 4);
    else if (it.part < 0) sym_finish<T, T>(it, a, ws.fac, tile, 4, 0);
    else {
        constexpr int PER = T / 8; float* out = reinterpret_cast<float*>(ws.split + (int64_t)it.part * PART);
#pragma unroll 2
        for (int z = 0; z < T * PER / 256; ++z) {
            const int r = z * (256 / PER) + threadIdx.x / PER; float v[8]; const int col = (threadIdx.x % PER) * 8; tile_row8<T>(tile, 4, r, col, v);
            *reinterpret_cast<f32x4*>(out + r * T + col) = f32x4{v[0], v[1], v[2], v[3]}; *reinterpret_cast<f32x4*>(out + r * T + col + 4) = f32x4{v[4], v[5], v[6], v[7]};
        }
    }
}
// A tile on or above the diagonal of a symmetric result, or its share of a split K axis
template <int T> __global__ __launch_bounds__(256, T == 128 ? 2 : 1) void ns_sym_kernel(Ws ws, SymArgs a) {
    __shared__ __attribute__((aligned(16))) char lds[Ring<T>::BYTES];
    const Item it = ws.sym[a.kind][blockIdx.x];
    sym_tile<T>(lds, it, ws, a);
}
// the shares of a tile, summed in order: 16 rows of a 128-tile or 32 of a 64-tile a workgroup (8 KB of each share)
template <int T> __device__ inline void reduce_tile(float* tile, const Item& it, const Ws& ws, const SymArgs& a, int r0) {
    constexpr int R = 2048 / T; const float* in = reinterpret_cast<const float*>(ws.split + (int64_t)it.part * PART) + r0 * T + threadIdx.x * 8;
    f32x4 v[2] = {};
#pragma unroll 8
    for (int k = 0; k < it.k1; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) v[h] += *reinterpret_cast<const f32x4*>(in + (int64_t)k * T * T + h * 4);
#pragma unroll
    for (int h = 0; h < 2; ++h) *reinterpret_cast<f32x4*>(tile + tile_at<T>(threadIdx.x / (T / 8), threadIdx.x % (T / 8) * 8 + h * 4)) = v[h];
    __syncthreads();
    sym_finish<T, R>(it, a, ws.fac, tile, 1, r0);
}
template <int T> __global__ __launch_bounds__(256) void ns_reduce_kernel(Ws ws, SymArgs a) {
    __shared__ __attribute__((aligned(16))) float tile[2048]; constexpr int SLABS = T * T / 2048;
    const Item it = ws.red[a.kind][blockIdx.x / SLABS];
    reduce_tile<T>(tile, it, ws, a, blockIdx.x % SLABS * (2048 / T));
}

// the shares of a whole short side (at most 64), and on to the product with it
__global__ __launch_bounds__(256) void ns_reduce_whole_kernel(Ws ws, SymArgs a) {
    __shared__ __attribute__((aligned(16))) char lds[16384 + 32768];
    const Item it = ws.red[a.kind][blockIdx.x]; float* tile = reinterpret_cast<float*>(lds); const float* in = reinterpret_cast<const float*>(ws.split + (int64_t)it.part * PART) + threadIdx.x * 8;
    f32x4 v[2][2] = {};
#pragma unroll 4
    for (int k = 0; k < it.k1; ++k)
#pragma unroll
        for (int z = 0; z < 2; ++z)
#pragma unroll
            for (int h = 0; h < 2; ++h) v[z][h] += *reinterpret_cast<const f32x4*>(in + (int64_t)k * 4096 + z * 2048 + h * 4);
#pragma unroll
    for (int z = 0; z < 2; ++z)
#pragma unroll
        for (int h = 0; h < 2; ++h) *reinterpret_cast<f32x4*>(tile + tile_at<64>(z * 32 + threadIdx.x / 8, threadIdx.x % 8 * 8 + h * 4)) = v[z][h];
    __syncthreads();
    sym_whole(lds + 16384, it, a, ws.fac, tile, 1);
}

enum { OUT_PAIR = 0, OUT_Y = 1, OUT_MUON = 2, OUT_BACK = 3 };
struct NnArgs { Slot l[2], r[2], e, out, x0; int nseg; float acc, ecoef, mid, decay; };      // value = acc * (mid * l0 r0 + l1 r1) + ecoef * e; one product: acc * l0 r0 + ecoef * e
template <int T, int DT, int OUT> __device__ inline void nn_tile(char* lds, double* red, const Item& it, const Ws& ws, const NnArgs& a, double* dots) {
    const Dims d = dims(it); const int kb = cdiv(it.m, 16), t = threadIdx.x;
    const Fac fac = ws.fac[it.mat]; const float facc = a.acc * fac.inv2;
    Seg seg[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) seg[s] = Seg{slot(it, d, a.r[s]) + (int64_t)it.tj * T * 4, slot(it, d, a.l[s]) + (int64_t)it.ti * T * d.arb, d.xrb, d.arb, 16 * d.xrb, 64};
    f32x16 c[2][2] = {};
    product<T, true>(lds, seg, a.nseg == 2 ? kb : 1 << 30, 0, a.nseg * kb, a.mid, c);
    // everything the epilogue reads is read before it writes anything: the loads are in flight together
    constexpr int N = T * T / 8 / 256; const char* E = slot(it, d, a.e); double dot = 0;
    f16x8 eh[N], el[N], xh[N], xl[N]; f32x4 P[N][2]; int64_t off[N];
    const Mat* M = &ws.mats[it.mat]; float* Y = OUT == OUT_MUON ? reinterpret_cast<float*>(M->y) : nullptr; int64_t ys = 0; bool rows = false;      // rows: the weight's rows as vectors
    if constexpr (OUT == OUT_MUON) { ys = M->ys; rows = M->yl == 1 && reinterpret_cast<uintptr_t>(Y) % 16 == 0 && ys % 4 == 0 && it.tj * T + T <= it.n; }
#pragma unroll
    for (int z = 0; z < N; ++z) {
        const int r = (z * 256 + t) / (T / 8), col = t % (T / 8) * 8, i = it.ti * T + r, j = it.tj * T + col;
        off[z] = pair_off(d.xrb, i, j);
        eh[z] = *reinterpret_cast<const f16x8*>(E + off[z]); el[z] = *reinterpret_cast<const f16x8*>(E + off[z] + LO);
        if constexpr (OUT == OUT_BACK) { xh[z] = *reinterpret_cast<const f16x8*>(slot(it, d, a.x0) + off[z]); xl[z] = *reinterpret_cast<const f16x8*>(slot(it, d, a.x0) + off[z] + LO); }
        if constexpr (OUT == OUT_MUON)
            if (rows && i < it.m) { P[z][0] = *reinterpret_cast<const f32x4*>(Y + i * ys + j); P[z][1] = *reinterpret_cast<const f32x4*>(Y + i * ys + j + 4); }
    }
    float* tile = reinterpret_cast<float*>(lds); tile_store<T>(tile, c);
#pragma unroll
    for (int z = 0; z < N; ++z) {
        const int r = (z * 256 + t) / (T / 8), col = t % (T / 8) * 8, i = it.ti * T + r, j = it.tj * T + col; float v[8], x[8];
        tile_row8<T>(tile, 4, r, col, v);
        unpack8(eh[z], el[z], x);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = facc * v[e] + a.ecoef * x[e];
        if constexpr (OUT == OUT_PAIR) store_pair8(slot(it, d, a.out) + off[z], v);
        else if constexpr (OUT == OUT_BACK) {                    // G in fp32, and this tile's share of <X0, G>
            unpack8(xh[z], xl[z], x);
#pragma unroll
            for (int e = 0; e < 8; ++e) dot += i < it.m ? (double)x[e] * (double)v[e] : 0.0;      // (rows behind the last may hold anything: 64-tiles of B and V do not cover 128)
            float* w = reinterpret_cast<float*>(slot(it, d, a.out) + i * d.xrb + (int64_t)j * 4);
            *reinterpret_cast<f32x4*>(w) = f32x4{v[0], v[1], v[2], v[3]}; *reinterpret_cast<f32x4*>(w + 4) = f32x4{v[4], v[5], v[6], v[7]};
        } else if (OUT == OUT_MUON && rows) {
            if (i < it.m)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) P[z][h][e] = a.decay * P[z][h][e] - M->alpha * ldexpf(v[h * 4 + e], -fac.q);
                    *reinterpret_cast<f32x4*>(Y + i * ys + j + h * 4) = P[z][h];
                }
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) *reinterpret_cast<f32x4*>(tile + tile_at<T>(r, col + h * 4)) = f32x4{v[h * 4], v[h * 4 + 1], v[h * 4 + 2], v[h * 4 + 3]};
        }
    }
    if constexpr (OUT == OUT_BACK) {
        dot = block_sum(dot, red);
        if (t == 0) dots[blockIdx.x] = dot;
    }
    if constexpr (OUT == OUT_Y || OUT == OUT_MUON) if (!rows) {  // element by element, neighbouring lanes along whichever axis is contiguous in the caller's memory
        const bool turn = M->ys == 1 && M->yl != 1; const int64_t yl = M->yl, yS = M->ys; char* y = M->y; const float alpha = M->alpha;
        __syncthreads();
#pragma unroll 1
        for (int b = 0; b < T * T / 256; b += 16) {
            float old[16]; int64_t o[16];
#pragma unroll
            for (int z = 0; z < 16; ++z) {
                const int q = (b + z) * 256 + t, r = turn ? q % T : q / T, col = turn ? q / T : q % T, i = it.ti * T + r, j = it.tj * T + col;
                o[z] = i < it.m && j < it.n ? i * yS + j * yl : -1;
                if constexpr (OUT == OUT_MUON) old[z] = o[z] >= 0 ? reinterpret_cast<float*>(y)[o[z]] : 0.f;
            }
#pragma unroll
            for (int z = 0; z < 16; ++z) {
                const int q = (b + z) * 256 + t, r = turn ? q % T : q / T, col = turn ? q / T : q % T;
                const float v = ldexpf(tile[tile_at<T>(r, col)], -fac.q);
                if (o[z] >= 0) { if constexpr (OUT == OUT_Y) st_el<DT>(y, o[z], v); else reinterpret_cast<float*>(y)[o[z]] = a.decay * old[z] - alpha * v; }
            }
        }
    }
}
// A tile of (symmetric m x m) x (m x n)
template <int T, int DT, int OUT> __global__ __launch_bounds__(256, T == 128 ? 2 : 1) void ns_nn_kernel(Ws ws, NnArgs a, double* dots) {
    __shared__ __attribute__((aligned(16))) char lds[Ring<T>::BYTES];
    const Item it = ws.nn[blockIdx.x];
    nn_tile<T, DT, OUT>(lds, reinterpret_cast<double*>(lds + 65536), it, ws, a, dots);      // (the epilogue's tile takes the first 64 KB)
}

// dX = (G - X0 <X0, G>) / |X|_F, or G / eps where the norm was clamped; G carries gscale / |dout|_F
template <int DT> __global__ __launch_bounds__(256) void ns_back_finish_kernel(Ws ws, const double* xpart, const double* dpart, const double* dots, Slot g, Slot x0, double gscale, double xscale, double eps) {
    __shared__ float lds[PK_ROWS * (PK_COLS + 1)]; __shared__ double red[4];
    const Item it = ws.pk[blockIdx.x]; const Mat M = ws.mats[it.mat];
    const int64_t xrb = (int64_t)M.np * 4; const int t = threadIdx.x; const bool turn = M.ys == 1 && M.yl != 1;
    f32x4 G[8]; f16x4 xh[8], xl[8];                              // (before the sums, which wait for memory too)
#pragma unroll
    for (int p = 0; p < 8; ++p) {
        const int i = it.ti * PK_ROWS + p * 8 + (t >> 5), j = it.tj * PK_COLS + (t & 31) * 4; const char* X0 = slot(M, x0) + pair_off(xrb, i, j);
        G[p] = *reinterpret_cast<const f32x4*>(slot(M, g) + i * xrb + (int64_t)j * 4); xh[p] = *reinterpret_cast<const f16x4*>(X0); xl[p] = *reinterpret_cast<const f16x4*>(X0 + LO);
    }
    const double norm = norm_of(M, xpart, red), dnorm = norm_of(M, dpart, red);
    double along = 0;
    for (int q = threadIdx.x; q < M.nnn; q += 256) along += dots[M.nn0 + q];
    along = block_sum(along, red) / xscale;
    // |dout| / (gscale |x|) as a factor in [1/2, 2) and a power of two: by itself it leaves fp32's range before dx does (G may be 2^14), and would turn zeros into NaN beyond it
    const bool clamped = norm <= eps; int ed, en; const double md = frexp(dnorm / gscale, &ed), mn = frexp(clamped ? eps : norm, &en);
    const float fg = (float)(md / mn), fx = clamped ? 0.f : (float)(along * (md / mn) / xscale); const int fe = ed - en;
#pragma unroll
    for (int p = 0; p < 8; ++p) {
        const int li = p * 8 + (t >> 5), lj = (t & 31) * 4, i = it.ti * PK_ROWS + li, j = it.tj * PK_COLS + lj;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float v = ldexpf(clamped ? G[p][e] * fg : G[p][e] * fg - ((float)xh[p][e] + (float)xl[p][e]) * fx, fe);
            if (turn) lds[li * (PK_COLS + 1) + lj + e] = v;
            else if (i < M.m && j + e < M.n) st_el<DT>(M.y, i * M.ys + (j + e) * M.yl, v);
        }
    }
    if (turn) {
        __syncthreads();
        for (int q = 0; q < PK_COLS / 4; ++q) {
            const int j = it.tj * PK_COLS + q * 4 + (t >> 6), i = it.ti * PK_ROWS + (t & 63);
            if (i < M.m && j < M.n) st_el<DT>(M.y, i * M.ys + j * M.yl, lds[(t & 63) * (PK_COLS + 1) + q * 4 + (t >> 6)]);
        }
    }
}

// ---- small matrices: a workgroup each, everything in LDS --------------------------------------------------------------------
// A call whose matrices all fit (short side MP = 32 or 64, pairs of X and A within 160 KB) is one launch: eight waves keep X in LDS from the first read to the result.  The launches of the
// tiled path cost 5 - 6 us each whatever the size; its 18 for a 64 x 64 matrix took 106 us.
// LDS rows are multiples of 256 bytes; row i's blocks of 64 are stored at block ^ (i & 3) and their chunks swizzled as the ring's, so that the products' row reads meet every bank.
template <int MT> struct Small {
    static constexpr int MP = MT * 32, TILES = MT * MT, KS = MT == 1 ? 4 : 2, AROW = MT == 1 ? 256 : MP * 4, AB = MT == 1 ? 12288 : MP * AROW, LDS = 163840;      // KS: waves that share a Gram tile's K axis
    __host__ __device__ static int blocks(int n) { return cdiv(n, 32) * 2; }                            // 16-column blocks of a row
    __host__ __device__ static int row(int n) { return cdiv(n, 64) * 256; }      // bytes of a row
    __host__ static bool fits(int m, int n) { return m <= MP && (int64_t)MP * row(n) + AB <= LDS; }
};
struct SmallArgs { int steps; float gram, poly, poly_e, apply, apply_e, last, last_e, decay; double eps, grow; MuonArgs mu; int dt_bytes; };
template <int N> struct SmallPack { Desc d[N]; };
template <int MT, int DT, int MUON, int N> __global__ __launch_bounds__(512) void ns_small_kernel(SmallPack<N> dp, Strides st, SmallArgs a) {
    using C = Small<MT>;
    __shared__ __attribute__((aligned(16))) char lds[C::LDS];
    const Desc& D = dp.d[N == 1 ? 0 : blockIdx.x]; const int b = N == 1 ? blockIdx.x : 0, m = D.m, n = D.n, nb = C::blocks(n), S = C::row(n);
    const int t = threadIdx.x, lane = t & 63, wv = t >> 6, lr = lane & 31, lk = lane >> 5;
    char *X = lds, *A = lds + C::MP * S; double* red = reinterpret_cast<double*>(A);
    const int64_t ys = D.tall ? 1 : n, yl = D.tall ? m : 1, ss = N == 1 ? st.xs : ys, sl = N == 1 ? st.xl : yl;
    const char* src = (const char*)D.x + (N == 1 ? st.xb * b * a.dt_bytes : 0); char* y = (char*)D.y + (int64_t)m * n * b * a.dt_bytes;
    const bool along = !(ss == 1 && sl != 1);                    // neighbouring lanes along the long side
    // X as fp32, each block of 16 columns where its pairs will be, and the norm
    double sum = 0; const int cols = nb * 16, all = C::MP * cols;
    for (int q0 = 0; q0 < all; q0 += 8 * 512) {
        float x[8], g[8]; int at[8]; int64_t o[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int q = q0 + u * 512 + t, i = along ? q / cols : q % C::MP, j = along ? q % cols : q / C::MP;
            at[u] = q < all ? i * S + (((j >> 4) ^ (i & 3)) << 6) + (j & 15) * 4 : -1; o[u] = q < all && i < m && j < n ? i * ss + j * sl : -1;      // (16 columns of fp32 take the 64 bytes of their block)
            x[u] = ld_el<DT>(src, o[u] >= 0 ? o[u] : 0); x[u] = o[u] >= 0 ? x[u] : 0.f;      // (no branch around a load, as in load_tile)
            if constexpr (MUON) { g[u] = reinterpret_cast<const float*>(D.d)[o[u] >= 0 ? o[u] : 0]; g[u] = o[u] >= 0 ? g[u] : 0.f; }
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            if constexpr (MUON) {
                x[u] = momentum_step(x[u], g[u], a.mu);
                if (o[u] >= 0) reinterpret_cast<float*>(const_cast<char*>(src))[o[u]] = x[u];
                x[u] = muon_u(x[u], g[u], a.mu);
            }
            if (at[u] >= 0) *reinterpret_cast<float*>(X + at[u]) = x[u];
            sum += (double)x[u] * (double)x[u];
        }
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    if (lane == 0) red[wv] = sum;
    __syncthreads();
    const double norm = sqrt(((red[0] + red[1]) + (red[2] + red[3])) + ((red[4] + red[5]) + (red[6] + red[7])));
    int fq = 0;
    if (norm <= a.eps && norm > 0) { const double room = 4.0 * a.eps / (norm * a.grow); if (room >= 2.0) fq = ilogb(room); }      // (as in ns_pack_kernel)
    const float inv2 = (float)ldexp(1.0, -2 * fq); int fe; const float f = (float)frexp(norm > 0 || norm != norm ? ldexp(SX, fq) / (norm <= a.eps ? a.eps : norm) : 0.0, &fe);
    for (int q = t; q < C::MP * nb; q += 512) {                  // a block of 16 columns a thread
        const int i = q / nb, blk = q % nb; char* p = X + i * S + ((blk ^ (i & 3)) << 6); f32x4 r[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) r[k] = *reinterpret_cast<const f32x4*>(p + k * 16);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float w[4]; f16x4 hi, lo;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = ldexpf(r[k][e], fe) * f;
            split4(w, hi, lo);
            *reinterpret_cast<f16x4*>(small_at(X, S, i, blk * 16 + k * 4, 0)) = hi; *reinterpret_cast<f16x4*>(small_at(X, S, i, blk * 16 + k * 4, 1)) = lo;
        }
    }
    __syncthreads();
    const int shares = nb >= 8 ? C::KS : 1;                      // (fewer blocks: joining shares costs more than it saves)
    const int tile = wv % C::TILES, ks = wv / C::TILES, i0 = tile / MT * 32, j0 = tile % MT * 32;
    for (int step = 0; step < a.steps; ++step) {
        const bool last = step == a.steps - 1;
        // A = X X^T: a 32 x 32 tile and a share of K a wave, three sums that do not wait for each other
        f32x16 c[3] = {};
        if (ks < shares) {
            for (int k = ks; k < nb; k += shares) {
                const f16x8 ah = small_row(X, S, i0 + lr, k, lk), al = small_row(X, S, i0 + lr, k, lk + 2), bh = small_row(X, S, j0 + lr, k, lk), bl = small_row(X, S, j0 + lr, k, lk + 2);
                c[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bh, c[0], 0, 0, 0); c[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al, bh, c[1], 0, 0, 0); c[2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bl, c[2], 0, 0, 0);
            }
            c[0] += c[1] + c[2];
            if (ks > 0)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    f32x4 w;
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = c[0][g * 4 + e];
                    *reinterpret_cast<f32x4*>(A + (((ks - 1) * C::TILES + tile) * 256 + g * 64 + lane) * 16) = w;
                }
        }
        if (shares > 1) {
            __syncthreads();
            if (ks == 0)
#pragma unroll
                for (int r = 1; r < C::KS; ++r)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const f32x4 w = *reinterpret_cast<const f32x4*>(A + (((r - 1) * C::TILES + tile) * 256 + g * 64 + lane) * 16);
#pragma unroll
                        for (int e = 0; e < 4; ++e) c[0][g * 4 + e] += w[e];
                    }
            __syncthreads();
        }
        auto write = [&](const f32x16& v) {                      // lane: row j0 + lr, registers: four neighbouring columns from i0 (A and B are symmetric)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float w[4] = {v[g * 4], v[g * 4 + 1], v[g * 4 + 2], v[g * 4 + 3]}; f16x4 hi, lo; split4(w, hi, lo); const int i = i0 + g * 8 + lk * 4;
                *reinterpret_cast<f16x4*>(small_at(A, C::AROW, j0 + lr, i, 0)) = hi; *reinterpret_cast<f16x4*>(small_at(A, C::AROW, j0 + lr, i, 1)) = lo;
            }
        };
        if (ks == 0) { c[0] *= a.gram; write(c[0]); }
        __syncthreads();
        // B = b A + c A A, in A's place
        f32x16 p[3] = {}; float E[16];
        if (ks == 0) {
#pragma unroll
            for (int k = 0; k < C::MP / 16; ++k) {
                const f16x8 ah = small_row(A, C::AROW, i0 + lr, k, lk), al = small_row(A, C::AROW, i0 + lr, k, lk + 2), bh = small_row(A, C::AROW, j0 + lr, k, lk), bl = small_row(A, C::AROW, j0 + lr, k, lk + 2);
                p[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bh, p[0], 0, 0, 0); p[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al, bh, p[1], 0, 0, 0); p[2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bl, p[2], 0, 0, 0);
            }
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int i = i0 + g * 8 + lk * 4;
                unpack4(*reinterpret_cast<const f16x4*>(small_at(A, C::AROW, j0 + lr, i, 0)), *reinterpret_cast<const f16x4*>(small_at(A, C::AROW, j0 + lr, i, 1)), E + g * 4);
            }
            p[0] += p[1] + p[2]; const float facc = a.poly * inv2;
#pragma unroll
            for (int e = 0; e < 16; ++e) p[0][e] = facc * p[0][e] + a.poly_e * E[e];
        }
        __syncthreads();
        if (ks == 0) write(p[0]);
        __syncthreads();
        // X <- a X + B X, a 32 x 32 tile a wave at a time, in place: a round's eight waves have read their columns before any of them writes; the last step leaves fp32
        const float facc = (last ? a.last : a.apply) * inv2, fe_ = last ? a.last_e : a.apply_e;
        for (int at = wv; at - wv < nb / 2 * MT; at += 8) {
            const bool mine = at < nb / 2 * MT; const int cg = at / MT, i = at % MT * 32 + lr;
            f16x8 xh[C::MP / 16], xl[C::MP / 16]; float e4[16];
            if (mine) {
                const int s = lane & 15, g4 = lane >> 4, blk = cg * 2 + (g4 & 1), chunk = (s & 3) >> 1;
#pragma unroll
                for (int k = 0; k < C::MP / 16; ++k) {
                    typedef __attribute__((address_space(3))) s16x4* p4; typedef short s16x8 __attribute__((ext_vector_type(8)));
                    s16x4 v[4];
#pragma unroll
                    for (int h = 0; h < 4; ++h) {                // rows 0..3 and 4..7 of the lane's eight; hi, lo
                        const int row = k * 16 + (g4 >> 1) * 8 + (h & 1) * 4 + (s >> 2);
                        v[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((p4)(X + row * S + ((blk ^ (row & 3)) << 6) + (((chunk + (h >> 1) * 2) ^ row_swizzle(row)) << 4) + (s & 1) * 8));
                    }
                    xh[k] = __builtin_bit_cast(f16x8, (s16x8)__builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7)); xl[k] = __builtin_bit_cast(f16x8, (s16x8)__builtin_shufflevector(v[2], v[3], 0, 1, 2, 3, 4, 5, 6, 7));
                }
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int j = cg * 32 + g * 8 + lk * 4;
                    unpack4(*reinterpret_cast<const f16x4*>(small_at(X, S, i, j, 0)), *reinterpret_cast<const f16x4*>(small_at(X, S, i, j, 1)), e4 + g * 4);
                }
            }
            __syncthreads();
            if (mine) {
                f32x16 d[3] = {};
#pragma unroll
                for (int k = 0; k < C::MP / 16; ++k) {
                    const f16x8 bh = small_row(A, C::AROW, i, k, lk), bl = small_row(A, C::AROW, i, k, lk + 2);
                    d[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(xh[k], bh, d[0], 0, 0, 0); d[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(xl[k], bh, d[1], 0, 0, 0); d[2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(xh[k], bl, d[2], 0, 0, 0);
                }
                d[0] += d[1] + d[2];
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int j = cg * 32 + g * 8 + lk * 4; float w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = facc * d[0][g * 4 + e] + fe_ * e4[g * 4 + e];
                    if (last) *reinterpret_cast<f32x4*>(X + i * S + (((j >> 4) ^ (i & 3)) << 6) + (j & 15) * 4) = f32x4{w[0], w[1], w[2], w[3]};
                    else { f16x4 hi, lo; split4(w, hi, lo); *reinterpret_cast<f16x4*>(small_at(X, S, i, j, 0)) = hi; *reinterpret_cast<f16x4*>(small_at(X, S, i, j, 1)) = lo; }
                }
            }
        }
        __syncthreads();
    }
    const bool turn = D.tall != 0;
    for (int q0 = 0; q0 < m * n; q0 += 8 * 512) {
        float old[8]; int64_t o[8]; int at[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int q = q0 + u * 512 + t, i = turn ? q % m : q / n, j = turn ? q / m : q % n;
            o[u] = q < m * n ? i * ys + j * yl : -1; at[u] = i * S + (((j >> 4) ^ (i & 3)) << 6) + (j & 15) * 4;
            if constexpr (MUON) old[u] = o[u] >= 0 ? reinterpret_cast<const float*>(y)[o[u]] : 0.f;
        }
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (o[u] >= 0) {
                const float v = ldexpf(*reinterpret_cast<const float*>(X + at[u]), -fq);
                if constexpr (MUON) reinterpret_cast<float*>(y)[o[u]] = a.decay * old[u] - D.alpha * v; else st_el<DT>(y, o[u], v);
            }
    }
}

// ---- host -------------------------------------------------------------------------------------------------------------------
// Bounds of what the iteration can meet, from the scalar polynomial on [0, s]: the iterates' singular values, B's, and by how much a step of the pullback can grow G
// grow, carry: a clamped matrix is carried at most 4 / (r grow) larger, the pullback's at most 4 / (r carry) (ns_pack_kernel)
struct Plan { bool ok = false; const char* why = ""; double grow = 1, carry = 1, growth[MD2_NS_MAX_STEPS + 1] = {}, s[MD2_NS_MAX_STEPS + 1] = {}, vgain[MD2_NS_MAX_STEPS] = {}; };
Plan ns_bounds(int steps, const double* co, bool back) {
    Plan P;
    if (steps < 1 || steps > MD2_NS_MAX_STEPS) { P.why = "steps must be in 1..16"; return P; }
    const double a = co[0], b = co[1], c = co[2];
    if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) { P.why = "the coefficients must be finite"; return P; }
    // with u = s^2 everything is a quadratic in u: its largest magnitude on [0, U] is at an end or at the vertex; the iterate's, s (a + b u + c u^2), where a + 3 b u + 5 c u^2 = 0
    auto most = [](double k0, double k1, double k2, double U) {
        double r = std::max(std::fabs(k0), std::fabs(k0 + U * (k1 + U * k2))); const double v = k2 != 0 ? -k1 / (2 * k2) : -1;
        return v > 0 && v < U ? std::max(r, std::fabs(k0 + v * (k1 + v * k2))) : r;
    };
    double lip[MD2_NS_MAX_STEPS], gain = 1.0, carry = 0.0; P.s[0] = 1.0;      // gain: how much larger than r = |X0| the iterate can be
    for (int k = 0; k < steps; ++k) {
        const double U = P.s[k] * P.s[k]; auto at = [&](double u) { return std::fabs(std::sqrt(u) * (a + u * (b + u * c))); };
        double top = at(U); const double disc = 9 * b * b - 20 * a * c, den = 10 * c;
        for (const double u : {den != 0 && disc >= 0 ? (-3 * b + std::sqrt(disc)) / den : -1.0, den != 0 && disc >= 0 ? (-3 * b - std::sqrt(disc)) / den : (b != 0 ? -a / (3 * b) : -1.0)})
            if (u > 0 && u < U) top = std::max(top, at(u));
        const double bm = most(0, b, c, U), up = most(a, b, c, U), L = std::max(up, most(a, 3 * b, 5 * c, U));
        P.s[k + 1] = top * 1.001; lip[k] = L * 1.001; P.vgain[k] = std::fabs(b) + 2 * std::fabs(c) * U;
        if (!(P.s[k + 1] <= 4.0) || !(bm <= 60.0)) { P.why = "these coefficients let a singular value grow past 4 (or b s^2 + c s^4 past 60)"; return P; }
        P.grow *= std::max(up, 1.0) * 1.001;
        if (gain > 0 && P.s[k] > 0) carry = std::max(carry, 4.0 * gain / P.s[k]);
        gain *= up * 1.001;
    }
    // The forward products hold a carried iterate of up to 4, whatever s[k] is; the pullback's S and V are scaled by s[k], so there a carried iterate, 2^q r gain, stays below s[k] as well.
    // (With coefficients that shrink singular values s[k] falls below 4 gain / grow, and S would pass f16's range.  With the default ones it does not: carry = grow.)
    P.carry = std::max(P.grow, carry);
    P.growth[steps] = 1.0;
    for (int k = steps - 1; k >= 0; --k) P.growth[k] = P.growth[k + 1] * std::max(lip[k], 1.0);
    if (back && !(P.growth[0] <= 8192.0)) { P.why = "the pullback of this many steps can grow a gradient past 8192 times its norm"; return P; }
    P.ok = true; return P;
}
double pow2_below(double v) { return std::exp2(std::min(std::floor(std::log2(v)), 40.0)); }      // (a scale; its bound is 0 where coefficients are)

int64_t up(int64_t v, int64_t q) { return (v + q - 1) / q * q; }
struct Layout { int64_t mats, sym[SYMS], red[SYMS], nn, pk, fac, part, split, buf, total; int64_t n_mats, n_sym[SYMS], n_red[SYMS], n_nn, n_pk; };

}  // namespace

struct NsProblem { std::vector<Desc> d; std::vector<Use> u; Strides st{}; int nX, nA, kinds; Cuts cuts{}; };      // u: [weight][kinds]

// Tiles and splits of a call's products, from its sizes alone, by a model of a launch.
// 128-tiles share a staged row between two waves (half the loads of 64-tiles, whose four waves split K instead) and are the faster ones where they fill the chip; a call with few tiles is over
// sooner in 64-tiles, and sooner still with its K axis cut.  Measured: a block of 16 K takes a 128-tile 0.4 us at two workgroups a CU and 0.5 alone, a 64-tile 0.14 (a step of its waves,
// 0.55, is four blocks) and 0.22 where the chip is full of them (their loads); a workgroup's way in and out is 4 us, which two 128-tiles a CU hide from each other; a cut K axis costs a launch of 5 us and its partial sums' way through memory.
// (512 x 4608, X X^T: 36 64-tiles in five pieces, which it takes, 14.9 us and 4.8 to join them, uncut 45; ten 128-tiles in 18 pieces 13.0 and 5.9.  B X: 144 128-tiles 19.3, 576 64-tiles 23.
// 512 x 2304, B X: 72 128-tiles 20, 288 64-tiles 15.)
// Of lists, whose items are of many lengths, it only ranks the choices: it gives the ResNet-18 and -50 networks' b A + c A A 9.5 and 25.8 us, where 64-tiles take 16.5 and 41.3 (an item that
// follows another on its CU costs more than 0.14 a block) and 128-tiles 28.2 and 44.4; their B X 44 and 98, measured 59.6 and 127; ResNet-50's X X^T 77 with the join, measured 86 + 12.7.
static constexpr int CUS = 256, MIN128 = 16, MIN64 = 16;
static constexpr double LAUNCH = 5.0, PART_US = 64.0 * 1024 * 2 / 5.0e6;
static double launch_us(int tile, int64_t items, int64_t work, int64_t longest, bool equal) {      // items, their K blocks in all, the longest one's; equal: they come in whole rounds
    const double rounds = (double)items / CUS, whole = equal && items > CUS ? std::ceil(rounds) : rounds;
    if (tile == 64) return std::max(std::max(longest * 0.14 + 4.0, equal ? std::ceil(rounds) * (longest * 0.14 + 4.0) : rounds * 4.0 + work * 0.14 / CUS), work * 0.22 / CUS + 4.0);
    return std::max(longest * (items <= CUS ? 0.5 : 0.8) + 4.0, (work * 0.4 / CUS + rounds * 2.0) * (rounds > 0 ? whole / rounds : 1.0));      // (0.8: beside another one)
}
static int64_t tri(int64_t m, int tile) { const int64_t t = (m + tile - 1) / tile; return t * (t + 1) / 2; }
static Layout ns_layout(NsProblem& p) {
    Layout L{}; p.u.assign(p.d.size() * p.kinds, Use{});
    int64_t buf = 0, split_max = 0; int widest = 0;
    for (const Desc& d : p.d) widest = std::max(widest, d.m);
    p.cuts.fuse = widest <= 64;
    for (int kind = 0; kind < p.kinds; ++kind) {
        int64_t part = 0; int most = 1, tile = 64, chunk = 1; double best = 1e30; const bool equal = p.d.size() == 1;
        for (const Desc& d : p.d) most = std::max(most, kblocks(kind, d.m, d.n));
        for (const int T : {128, 64})
            for (int c = most; T == 64 || !p.cuts.fuse; c = std::max(T == 128 ? MIN128 : MIN64, std::min(c - 1, c * 7 / 8))) {
                int64_t items = 0, parts = 0, work = 0, longest = 0;
                for (const Desc& d : p.d) {
                    const int kb = kblocks(kind, d.m, d.n), sp = cdiv(kb, c); const int64_t t = d.batch * tri(d.m, T);
                    items += t * sp; work += t * kb; longest = std::max<int64_t>(longest, cdiv(kb, sp)); if (sp > 1) parts += t * sp;
                }
                const double us = launch_us(T, items, work, longest, equal) + (parts ? LAUNCH : 0) + parts * PART_US / (T == 128 ? 1 : 4);
                if (us < best) { best = us; tile = T; chunk = c; }
                if (c <= (T == 128 ? MIN128 : MIN64)) break;
            }
        p.cuts.sym[kind] = Cut{tile, chunk};
        for (size_t i = 0; i < p.d.size(); ++i) {
            const Desc& d = p.d[i]; Use& u = p.u[i * p.kinds + kind]; const int kb = kblocks(kind, d.m, d.n), split = cdiv(kb, cdiv(kb, cdiv(kb, chunk))); const int64_t tiles = d.batch * tri(d.m, tile);
            u = Use{(int)L.n_sym[kind], (int)L.n_red[kind], (int)part};
            L.n_sym[kind] += tiles * split;
            if (split > 1) { L.n_red[kind] += tiles; part += tiles * split * (tile * tile * 4 / PART); }
        }
        split_max = std::max(split_max, part);
    }
    double nn[2];
    for (const int T : {128, 64}) {
        int64_t items = 0, work = 0, longest = 0; const int seg = p.kinds == SYMS ? 2 : 1;
        for (const Desc& d : p.d) { const int64_t t = (int64_t)d.batch * cdiv(d.m, T) * cdiv(d.n, T), kb = seg * cdiv(d.m, 16); items += t; work += t * kb; longest = std::max(longest, kb); }
        nn[T == 64] = launch_us(T, items, work, longest, p.d.size() == 1);
    }
    p.cuts.nn_tile = !p.cuts.fuse && nn[0] <= nn[1] ? 128 : 64;
    for (Desc& d : p.d) {
        const int64_t mt = cdiv(d.m, PAD), nt = cdiv(d.n, PAD);
        d.first = (int)L.n_mats; d.nn0 = (int)L.n_nn; d.pk0 = (int)L.n_pk;
        d.ws0 = buf; d.ws1 = (p.nX * mt * nt + p.nA * mt * mt) * (int64_t)PAD * PAD * 4;
        L.n_mats += d.batch; L.n_nn += (int64_t)cdiv(d.m, p.cuts.nn_tile) * cdiv(d.n, p.cuts.nn_tile) * d.batch; L.n_pk += mt * (PAD / PK_ROWS) * nt * (PAD / PK_COLS) * d.batch;
        buf += d.ws1 * d.batch;
    }
    int64_t at = 0;
    auto take = [&](int64_t bytes) { const int64_t r = at; at = up(at + bytes, 256); return r; };
    L.mats = take(L.n_mats * sizeof(Mat));
    for (int k = 0; k < SYMS; ++k) { L.sym[k] = take(L.n_sym[k] * sizeof(Item)); L.red[k] = take(L.n_red[k] * sizeof(Item)); }
    L.nn = take(L.n_nn * sizeof(Item)); L.pk = take(L.n_pk * sizeof(Item)); L.fac = take(L.n_mats * sizeof(Fac));
    L.part = take((2 * L.n_pk + L.n_nn) * sizeof(double)); L.split = take(split_max * PART); L.buf = take(buf); L.total = at;
    return L;
}
static bool fits(int64_t batch, int64_t rows, int64_t cols) {      // (a matrix may have 2^31 elements: offsets of elements are 64-bit; the work items are counted in check_total)
    return rows > 0 && cols > 0 && batch > 0 && rows <= (1 << 20) && cols <= (1 << 20) && rows * cols <= (1ll << 31) && batch <= (1 << 20);
}
static int64_t check_total(const Layout& L) {      // (a launch has fewer than 2^32 threads: 2^24 workgroups of 256)
    for (int k = 0; k < SYMS; ++k) if (L.n_sym[k] >= (1ll << 24) || L.n_red[k] * 8 >= (1ll << 24)) return -1;
    return (L.n_nn < (1ll << 24) && L.n_pk < (1ll << 24) - 1024 && L.n_mats < (1ll << 24)) ? L.total : -1;
}

static Desc make_desc(const NsMatrices& q) {
    Desc d{}; const bool tall = q.rows > q.cols;
    d.x = q.x; d.d = q.d; d.y = q.y; d.m = (int)std::min(q.rows, q.cols); d.n = (int)std::max(q.rows, q.cols); d.batch = (int)q.batch;
    d.alpha = q.alpha; d.tall = tall;
    return d;
}
static void slots_of(int kind, int steps, NsProblem& p) {
    int &nX = p.nX, &nA = p.nA; p.kinds = kind == NS_BACKWARD ? SYMS : 2;
    if (kind == NS_BACKWARD) { nX = steps + 2; nA = 2 * steps + 2; }      // every iterate and two G | every A, every B, S, V
    else { nX = 2; nA = 2; }                                             // X twice | A, B
}
// 1 or 2: every matrix of a forward or Muon call fits Small<1> or Small<2>; 0: the tiled path
static int ns_small(int kind, const std::vector<Desc>& d) {
    if (kind == NS_BACKWARD) return 0;
    bool one = true, two = true;
    for (const Desc& q : d) { one = one && Small<1>::fits(q.m, q.n); two = two && Small<2>::fits(q.m, q.n); }
    return one ? 1 : two ? 2 : 0;
}
template <int MT, int DT> static void small_launch(int kind, const NsProblem& p, const SmallArgs& a, hipStream_t s) {
    if (kind == NS_MUON)
        for (size_t i = 0; i < p.d.size(); i += MUON_DESCS) {
            SmallPack<MUON_DESCS> dp; const int n = (int)std::min<size_t>(MUON_DESCS, p.d.size() - i);
            for (int k = 0; k < n; ++k) dp.d[k] = p.d[i + k];
            hipLaunchKernelGGL((ns_small_kernel<MT, NS_F32, 1, MUON_DESCS>), dim3(n), dim3(512), 0, s, dp, p.st, a);
        }
    else { SmallPack<1> dp; dp.d[0] = p.d[0]; hipLaunchKernelGGL((ns_small_kernel<MT, DT, 0, 1>), dim3(p.d[0].batch), dim3(512), 0, s, dp, p.st, a); }
}
int64_t ns_workspace(int kind, int steps, const NsMatrices* q, int count) {
    if (steps < 1 || steps > MD2_NS_MAX_STEPS) return -1;
    NsProblem p; slots_of(kind, steps, p);
    for (int i = 0; i < count; ++i) { if (!fits(q[i].batch, q[i].rows, q[i].cols)) return -1; p.d.push_back(make_desc(q[i])); }
    if (ns_small(kind, p.d)) return 256;                         // (none is used; a caller's buffer is never empty)
    std::stable_sort(p.d.begin(), p.d.end(), [](const Desc& a, const Desc& b) { return a.m > b.m; });
    return check_total(ns_layout(p));
}

int ns_tiles(int kind, int steps, const NsMatrices* q, int count, int32_t side[5], int32_t pieces[5]) {
    for (int k = 0; k < 5; ++k) side[k] = pieces[k] = 0;
    if (ns_workspace(kind, steps, q, count) < 0) return -1;
    NsProblem p; slots_of(kind, steps, p);
    for (int i = 0; i < count; ++i) p.d.push_back(make_desc(q[i]));
    if (ns_small(kind, p.d)) return 0;
    std::stable_sort(p.d.begin(), p.d.end(), [](const Desc& a, const Desc& b) { return a.m > b.m; });
    ns_layout(p);
    for (int k = 0; k < p.kinds; ++k) {
        if (p.cuts.fuse && (k == POLY || k == SYM_V)) continue;      // (done by X X^T's and S's workgroups)
        const int kb = kblocks(k, p.d[0].m, p.d[0].n); side[k] = p.cuts.sym[k].tile; pieces[k] = cdiv(kb, cdiv(kb, cdiv(kb, p.cuts.sym[k].chunk)));
    }
    side[4] = p.cuts.nn_tile; pieces[4] = 1;
    return 0;
}

template <int DT> static void ns_launch(int kind, NsProblem& p, const Layout& L, char* base, const NsOptions& o, const Plan& P, hipStream_t s) {
    Ws ws; ws.mats = (Mat*)(base + L.mats); for (int k = 0; k < SYMS; ++k) { ws.sym[k] = (Item*)(base + L.sym[k]); ws.red[k] = (Item*)(base + L.red[k]); } ws.nn = (Item*)(base + L.nn); ws.pk = (Item*)(base + L.pk); ws.fac = (Fac*)(base + L.fac); ws.part = (double*)(base + L.part); ws.split = base + L.split; ws.buf = base + L.buf;
    const int steps = o.steps;
    if (const int mt = ns_small(kind, p.d)) {
        const double a = o.coef[0], b = o.coef[1], c = o.coef[2];
        SmallArgs q{steps, (float)(SA / (SX * SX)), (float)(c * SB / (SA * SA)), (float)(b * SB / SA), (float)(1.0 / SB), (float)a, (float)(1.0 / (SB * SX)), (float)(a / SX), (float)(1.0 - o.lr * o.weight_decay),
                    o.eps, P.grow, MuonArgs{(float)o.momentum, (float)(1.0 - o.momentum), o.grad_scale, o.nesterov}, DT == NS_F32 ? 4 : 2};
        if (mt == 1) small_launch<1, DT>(kind, p, q, s); else small_launch<2, DT>(kind, p, q, s);
        return;
    }
    const dim3 blk(256), pk((unsigned)L.n_pk), nn((unsigned)L.n_nn);
#define NN(dt, out) do { if (p.cuts.nn_tile == 128) hipLaunchKernelGGL((ns_nn_kernel<128, dt, out>), nn, blk, 0, s, ws, f, dots); \
                         else hipLaunchKernelGGL((ns_nn_kernel<64, dt, out>), nn, blk, 0, s, ws, f, dots); } while (0)
    auto sym = [&](const SymArgs& a) {
        if (p.cuts.sym[a.kind].tile == 128) hipLaunchKernelGGL((ns_sym_kernel<128>), dim3((unsigned)L.n_sym[a.kind]), blk, 0, s, ws, a);
        else hipLaunchKernelGGL((ns_sym_kernel<64>), dim3((unsigned)L.n_sym[a.kind]), blk, 0, s, ws, a);
        if (!L.n_red[a.kind]) return;
        if (a.fuse) { hipLaunchKernelGGL(ns_reduce_whole_kernel, dim3((unsigned)L.n_red[a.kind]), blk, 0, s, ws, a); return; }
        if (p.cuts.sym[a.kind].tile == 128) hipLaunchKernelGGL((ns_reduce_kernel<128>), dim3((unsigned)L.n_red[a.kind] * 8), blk, 0, s, ws, a);
        else hipLaunchKernelGGL((ns_reduce_kernel<64>), dim3((unsigned)L.n_red[a.kind] * 2), blk, 0, s, ws, a);
    };
    const MuonArgs mu{(float)o.momentum, (float)(1.0 - o.momentum), o.grad_scale, o.nesterov};
    const double a = o.coef[0], b = o.coef[1], c = o.coef[2];
    const bool back = kind == NS_BACKWARD;
    double *xpart = ws.part, *dpart = ws.part + L.n_pk, *dots = ws.part + 2 * L.n_pk;
    auto sg = [&](int k) { return pow2_below(16384.0 / P.growth[k]); };                 // scale of dL/dX_k (of dout / |dout|: at most growth[k])
    if (kind == NS_MUON) {
        for (size_t i = 0; i < p.d.size(); i += MUON_DESCS) {
            DescPack<MUON_DESCS, 2> dp; const int n = (int)std::min<size_t>(MUON_DESCS, p.d.size() - i); const int64_t next = i + n < p.d.size() ? p.d[i + n].pk0 : L.n_pk;
            for (int k = 0; k < n; ++k) { dp.d[k] = p.d[i + k]; for (int u = 0; u < 2; ++u) dp.u[k][u] = p.u[(i + k) * 2 + u]; }
            hipLaunchKernelGGL((ns_start_kernel<NS_F32, SRC_MUON, MUON_DESCS, 2>), dim3((unsigned)(n + next - p.d[i].pk0)), blk, 0, s, dp, n, n, (int)L.n_pk, p.st, p.cuts, ws, mu);
        }
        hipLaunchKernelGGL((ns_pack_kernel<NS_F32, SRC_MUON>), pk, blk, 0, s, ws, mu, SX, o.eps, P.grow, 0, 0.0);
    } else {
        const int tables = std::min(p.d[0].batch, 1024); const dim3 both(pk.x, back ? 2 : 1), start(pk.x + tables, both.y);
        if (back) { DescPack<1, 4> dp; dp.d[0] = p.d[0]; for (int u = 0; u < 4; ++u) dp.u[0][u] = p.u[u]; hipLaunchKernelGGL((ns_start_kernel<DT, SRC_X, 1, 4>), start, blk, 0, s, dp, 1, tables, (int)L.n_pk, p.st, p.cuts, ws, mu); }
        else { DescPack<1, 2> dp; dp.d[0] = p.d[0]; for (int u = 0; u < 2; ++u) dp.u[0][u] = p.u[u]; hipLaunchKernelGGL((ns_start_kernel<DT, SRC_X, 1, 2>), start, blk, 0, s, dp, 1, tables, (int)L.n_pk, p.st, p.cuts, ws, mu); }
        hipLaunchKernelGGL((ns_pack_kernel<DT, SRC_X>), both, blk, 0, s, ws, mu, SX, o.eps, back ? P.carry : P.grow, steps, back ? sg(steps) : 0.0);
    }
    const int nX = p.nX;
    auto X = [&](int k) { return Slot{back ? k : (k & 1), 0}; };
    auto A = [&](int k) { return Slot{nX, back ? 2 * k : 0}; };
    auto B = [&](int k) { return Slot{nX, back ? 2 * k + 1 : 1}; };
    for (int k = 0; k < steps; ++k) {
        SymArgs g{}; g.l[0] = g.r[0] = X(k); g.e = g.out = A(k); g.nseg = 1; g.kind = GRAM; g.acc = (float)(SA / (SX * SX));
        g.fuse = p.cuts.fuse; g.then = B(k); g.acc2 = (float)(c * SB / (SA * SA)); g.ecoef2 = (float)(b * SB / SA);
        sym(g);
        SymArgs q{}; q.l[0] = q.r[0] = q.e = A(k); q.out = B(k); q.nseg = 1; q.kind = POLY; q.have_e = 1; q.acc = (float)(c * SB / (SA * SA)); q.ecoef = (float)(b * SB / SA);
        if (!p.cuts.fuse) sym(q);
        if (back && k == steps - 1) break;
        NnArgs f{}; f.l[0] = B(k); f.r[0] = f.e = X(k); f.out = X(k + 1); f.nseg = 1;
        if (k < steps - 1) { f.acc = (float)(1.0 / SB); f.ecoef = (float)a; NN(NS_F32, OUT_PAIR); }
        else {
            f.acc = (float)(1.0 / (SB * SX)); f.ecoef = (float)(a / SX); f.decay = (float)(1.0 - o.lr * o.weight_decay);
            if (kind == NS_MUON) NN(NS_F32, OUT_MUON);
            else NN(DT, OUT_Y);
        }
    }
    if (!back) return;
    const Slot G[2] = {Slot{steps, 0}, Slot{steps + 1, 0}}; const Slot S{nX, 2 * steps}, V{nX, 2 * steps + 1};
    int cur = 0;
    for (int k = steps - 1; k >= 0; --k, cur ^= 1) {
        const double gin = sg(k + 1), gout = sg(k), sbound = 2 * P.growth[k + 1] * P.s[k];
        const double ss = pow2_below(16384.0 / sbound), sv = pow2_below(16384.0 / (sbound * P.vgain[k]));
        SymArgs q{}; q.l[0] = G[cur]; q.r[0] = X(k); q.l[1] = X(k); q.r[1] = G[cur]; q.e = q.out = S; q.nseg = 2; q.kind = SYM_S; q.acc = (float)(ss / (gin * SX));
        q.fuse = p.cuts.fuse; q.with = A(k); q.then = V; q.acc2 = (float)(c * sv / (ss * SA)); q.ecoef2 = (float)(b * sv / ss);
        sym(q);
        SymArgs v{}; v.l[0] = S; v.r[0] = A(k); v.l[1] = A(k); v.r[1] = S; v.e = S; v.out = V; v.nseg = 2; v.kind = SYM_V; v.have_e = 1; v.acc = (float)(c * sv / (ss * SA)); v.ecoef = (float)(b * sv / ss);
        if (!p.cuts.fuse) sym(v);
        NnArgs f{}; f.l[0] = B(k); f.r[0] = f.e = G[cur]; f.l[1] = V; f.r[1] = X(k); f.out = G[cur ^ 1]; f.x0 = X(0); f.nseg = 2;
        f.mid = (float)(sv * SX / (SB * gin)); f.acc = (float)(gout / (sv * SX)); f.ecoef = (float)(a * gout / gin);
        if (k > 0) NN(NS_F32, OUT_PAIR);
        else NN(NS_F32, OUT_BACK);
    }
    hipLaunchKernelGGL((ns_back_finish_kernel<DT>), pk, blk, 0, s, ws, xpart, dpart, dots, G[cur], X(0), sg(0), SX, o.eps);
#undef NN
}

// (any fp32 norm over any fp32 eps, and the carry of a clamped matrix, stay far inside the range of doubles)
static const char* const kEps = "eps must be positive and at most 3.4e38";
static bool eps_ok(double eps) { return eps > 0 && eps <= 3.4e38; }
const char* ns_check(int steps, const double* co, double eps) {
    if (!eps_ok(eps)) return kEps;
    const Plan P = ns_bounds(steps, co, false);
    return P.ok ? nullptr : P.why;
}
// does memory of so many bytes share any with what `st` reaches from p? | the contiguous result?
static bool overlaps(const void* a, __int128 bytes, const NsMatrices& q, const void* p, const int64_t st[3], int el) {
    const __int128 a0 = (__int128)(uintptr_t)a, p0 = (__int128)(uintptr_t)p;
    const __int128 p1 = p0 + ((__int128)(q.batch - 1) * st[0] + (__int128)(q.rows - 1) * st[1] + (__int128)(q.cols - 1) * st[2] + 1) * el;
    return a0 < p1 && p0 < a0 + bytes;
}
static bool overlaps(const NsMatrices& q, const void* p, const int64_t st[3], int el) { return overlaps(q.y, (__int128)q.batch * q.rows * q.cols * el, q, p, st, el); }
int ns_run(int kind, int dtype, const NsMatrices* q, int count, const NsOptions& o, void* wsp, int64_t ws_bytes, hipStream_t s, const char** why) {
    if (!eps_ok(o.eps)) { *why = kEps; return 2; }
    const Plan P = ns_bounds(o.steps, o.coef, kind == NS_BACKWARD);
    if (!P.ok) { *why = P.why; return 2; }
    const int el = dtype == NS_F32 ? 4 : 2;
    NsProblem p; slots_of(kind, o.steps, p);
    for (int i = 0; i < count; ++i) {
        const NsMatrices& m = q[i];
        if (!m.x || !m.y || (kind != NS_FORWARD && !m.d)) { *why = "null pointer"; return 2; }
        if (!fits(m.batch, m.rows, m.cols)) { *why = "sizes must be positive, a side at most 2^20, a matrix at most 2^31 elements, a batch at most 2^20"; return 2; }
        if (((uintptr_t)m.x | (uintptr_t)m.d | (uintptr_t)m.y) % el) { *why = "a pointer is not aligned to its elements"; return 2; }
        for (int k = 0; k < 3; ++k) if (m.xs[k] < 0 || m.ds[k] < 0) { *why = "negative stride"; return 2; }
        // (one matrix may be written before another is read)
        if (kind != NS_MUON && (overlaps(m, m.x, m.xs, el) || (kind == NS_BACKWARD && overlaps(m, m.d, m.ds, el)))) { *why = "the result overlaps an input"; return 2; }
        p.d.push_back(make_desc(m));
    }
    if (kind != NS_MUON) { const bool tall = p.d[0].tall; const int64_t *x = q[0].xs, *d = q[0].ds; p.st = Strides{x[0], x[tall ? 2 : 1], x[tall ? 1 : 2], d[0], d[tall ? 2 : 1], d[tall ? 1 : 2]}; }
    std::stable_sort(p.d.begin(), p.d.end(), [](const Desc& a, const Desc& b) { return a.m > b.m; });      // the longest work items first
    Layout L{}; L.total = 256;
    if (!ns_small(kind, p.d)) { L = ns_layout(p); if (check_total(L) < 0) { *why = "too many matrices"; return 2; } }
    if (!wsp || (uintptr_t)wsp % 256 || ws_bytes < L.total) { *why = "the workspace is missing, too small or not aligned to 256 bytes"; return 2; }
    if (!ns_small(kind, p.d))                                    // (which uses none)
        for (int i = 0; i < count; ++i) {
            const NsMatrices& m = q[i]; const int64_t ys[3] = {m.rows * m.cols, m.cols, 1};
            if (overlaps(wsp, L.total, m, m.x, m.xs, el) || overlaps(wsp, L.total, m, m.y, ys, el) || (m.d && overlaps(wsp, L.total, m, m.d, m.ds, el))) { *why = "the workspace overlaps an input or a result"; return 2; }
        }
    if (dtype == NS_F32) ns_launch<NS_F32>(kind, p, L, (char*)wsp, o, P, s);
    else if (dtype == NS_BF16) ns_launch<NS_BF16>(kind, p, L, (char*)wsp, o, P, s);
    else ns_launch<NS_F16>(kind, p, L, (char*)wsp, o, P, s);
    return 0;
}

}  // namespace md2
