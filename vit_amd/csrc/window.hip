// Attention with a sliding window and sinks over long token sequences: forward and backward.
//
//   visible(i, j) = (|i - j| <= w  or  j < S  or  w < 0)  and  (not causal or j <= i)  and  i, j < length of the sequence
//   P_ij = exp(scale q_i . k_j - lse_i),  o_i = sum_j P_ij v_j        over the visible j; a row that sees nothing is zero
//   D_i = do_i . o_i,  dS_ij = P_ij (do_i . v_j - D_i)
//   dq_i = scale sum_j dS_ij k_j,  dk_j = scale sum_i dS_ij q_i,  dv_j = sum_i P_ij do_i   (dk, dv: over the group's heads)
//
// Only tiles that hold a visible pair are touched: a block of queries walks its window's key tiles and the sinks' tiles
// before (or after) them.  Scores are made transposed, S^T[key][query] = K Q^T by 32 x 32 x 16 MFMA, so a lane owns one
// query: the running maximum and sum are one value a lane, and the probability tile is already the B operand of
// O^T += V^T P^T (the order of the contraction's 16 keys is the accumulator's own; V^T fragments come from the row-major
// V tile in LDS by transpose reads in that same order).  Nothing of size N x N exists and nothing is summed by atomics:
// the backward makes the scores twice (queries' kernel, keys' kernel).  Sums, maxima and the softmax are fp32; with bf16
// inputs P and dS are rounded to bf16 as operands of their MFMA, each once; in calls of few scores what that took is
// multiplied as well.
#include <algorithm>
#include <type_traits>
#include "common.h"

namespace vitk {

typedef __attribute__((ext_vector_type(16))) float f32x16;

// D(32x32) += A(32x16) B(16x32).  Frag convention here: lane l holds row (A) / column (B) l & 31, k = 8 (l >> 5) + e.
// D: register r of lane l is row 8 (r >> 2) + 4 (l >> 5) + (r & 3), column l & 31.  The fp32 form feeds element e of both
// halves to step e: the same permutation of k on both sides.
__device__ __forceinline__ f32x16 mma32(const Frag<__bf16>& a, const Frag<__bf16>& b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, b.v, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma32(const Frag<float>& a, const Frag<float>& b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[e], b.v[e], c, 0, 0, 0);
    return c;
}
// accumulator rows 16 s .. 16 s + 15 as a B fragment: element e is row 16 s + 8 (e >> 2) + 4 (l >> 5) + (e & 3)
template <typename T> __device__ __forceinline__ void acc_frag(Frag<T>& f, const f32x16& a, int s) {
#pragma unroll
    for (int e = 0; e < 8; ++e) frag_set_f(f, e, a[8 * s + e]);
}
// what the rounding to acc_frag's bf16 took
__device__ __forceinline__ void rest_frag(Frag<__bf16>& r, const Frag<__bf16>& f, const f32x16& a, int s) {
#pragma unroll
    for (int e = 0; e < 8; ++e) frag_set_f(r, e, a[8 * s + e] - frag_get_f(f, e));
}
// LDS image of a tile: rows of CPR 16-byte chunks without padding (what the asynchronous loads can write: 64 consecutive
// chunks an instruction); chunk c of row r sits at place c ^ swz(r).  The 64 banks hold 16 chunks.  A row fragment reads
// one chunk of each row: over 16 rows swz (with the row's own offset where a row is shorter than the banks) takes every
// value.  A transpose read takes 4 chunks of each of 4 rows: its low two bits stay among those 4, its upper bits (or the
// row's offset) send the 4 rows to different quarters of the banks.  With swz = r & 7, two thirds of the LDS time at 128
// wide heads were conflicts.
template <typename T, int DP> struct WCfg {
    static constexpr int EPC = 16 / sizeof(T);          // elements of a 16-byte chunk
    static constexpr int CPR = DP / EPC;                // chunks of a row
    static constexpr int LD = DP + EPC;                 // row stride of the results' image (put_rows)
    static __device__ __forceinline__ int swz(int r) {
        return CPR % 16 == 0 ? ((r & 3) << 2) | ((r >> 2) & 3) : (CPR % 8 == 0 ? ((r & 2) << 1) | ((r >> 2) & 3) : (r >> 2) & 3);
    }
};
// the A fragment that goes with acc_frag: columns col0 + (l & 31) of an image, rows row0 + the order above (row0 % 16 == 0).
// bf16: transpose reads -- lane 4 q + p of 16 supplies row q, columns 4 p .. 4 p + 3, and receives column l & 15 of the 4
// rows; needs every lane of the wave.
template <int DP> __device__ __forceinline__ void col_frag32(Frag<__bf16>& f, const __bf16* img, int row0, int col0, int lane) {
    using C = WCfg<__bf16, DP>;
    const int i = lane & 15, q = i >> 2, p = i & 3, r = 4 * (lane >> 5) + q;
    const int c = (col0 / 8 + 2 * ((lane >> 4) & 1) + (p >> 1)) ^ C::swz(r);
    const __bf16* a = img + (row0 + r) * DP + 8 * c + 4 * (p & 1);
    const __bf16* b = img + (row0 + r + 8) * DP + 8 * (c ^ 2) + 4 * (p & 1);             // swz(r + 8) = swz(r) ^ 2 here (r < 8)
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(uintptr_t)a);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(uintptr_t)b);
    const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    f.v = __builtin_bit_cast(bf16x8, v);
}
template <int DP> __device__ __forceinline__ void col_frag32(Frag<float>& f, const float* img, int row0, int col0, int lane) {
    using C = WCfg<float, DP>;
    const int cc = lane & 31;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int r = 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
        f.v[e] = img[(row0 + r) * DP + 4 * ((col0 / 4 + cc / 4) ^ C::swz(r)) + (cc & 3)];
    }
}
// row row0 + (l & 31), elements 16 kk + 8 (l >> 5) + e (row0 % 32 == 0)
template <int DP> __device__ __forceinline__ void row_frag32(Frag<__bf16>& f, const __bf16* img, int row0, int kk, int lane) {
    const int r = lane & 31;
    frag_load(f, img + (row0 + r) * DP + 8 * ((2 * kk + (lane >> 5)) ^ WCfg<__bf16, DP>::swz(r)));
}
template <int DP> __device__ __forceinline__ void row_frag32(Frag<float>& f, const float* img, int row0, int kk, int lane) {
    const int r = lane & 31, s = WCfg<float, DP>::swz(r), c = 4 * kk + 2 * (lane >> 5);
    const float* a = img + (row0 + r) * DP;
    const f32x4 x = *reinterpret_cast<const f32x4*>(a + 4 * (c ^ s)), y = *reinterpret_cast<const f32x4*>(a + 4 * ((c + 1) ^ s));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        f.v[e] = x[e];
        f.v[4 + e] = y[e];
    }
}

// part 0: the finite values, 0 for the others; 1: 1 for +inf and NaN, else 0; 2: 1 for -inf and NaN, else 0
__device__ __forceinline__ void value_part(Frag<float>& f, int part) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float x = f.v[e];
        const bool finite = fabsf(x) < INFINITY;
        f.v[e] = part == 0 ? (finite ? x : 0.f) : (finite || x == (part == 1 ? -INFINITY : INFINITY) ? 0.f : 1.f);
    }
}
__device__ __forceinline__ void value_part(Frag<__bf16>& f, int part) {
    const s16x8 x = __builtin_bit_cast(s16x8, f.v), beyond = (x & (short)0x7f80) == (short)0x7f80;      // all bits where not finite
    s16x8 y = x & ~beyond;
    if (part) y = beyond & (x != (short)(part == 1 ? 0xff80 : 0x7f80)) & (short)0x3f80;
    f.v = __builtin_bit_cast(bf16x8, y);
}

struct View {                     // element (b, n, h, d) at b*sb + n*sn + h*sh + d
    const void* p;
    long sb, sn, sh;
};
struct WindowParams {
    View q, k, v, dout;           // dout: backward
    const void* o;                // backward: the forward's output, [B][N][Hq][dh]
    void* o_lo;                   // bf16, or NULL: what rounding took from o, rounded itself; the forward writes it, D reads it
    void *out, *dk, *dv;          // out: o in the forward, dq in the queries' backward kernel; all [B][N][H][dh]
    float* lse;                   // [B][Hq][N]: log2 of the softmax sum, maximum included; +inf where a row sees nothing
    float* delta;                 // [B][Hq][N]: D_i, written by the queries' kernel for the keys' kernel
    int* far;                     // the same way, [B][Hq][groups of 32 rows]: whether one of them has a far log-sum
    float* shift;                 // [B][Hq][N]: in such groups, what the rows' exponents lack
    float* part;                  // sinks' partial sums [B*Hk][key tiles][chunks][dk, dv][DP][32] fp32
    const int* lengths;           // [B] or NULL
    int B, N, Hq, Hk, G, dh;
    int w, S, causal;
    int tiles;                    // query tiles / key tiles of a sequence
    int key0;                     // keys' kernel: first key (the sinks before it have their own launch)
    int heavy;                    // keys' kernel: how many of a sequence's tiles, the first ones, hold sinks
    int chunks, per_chunk;        // sinks' launch: query tiles are dealt to `chunks` workgroups
    // order of the pieces of work: tiles within a (sequence, key head), or (by_tile) all sequences' and heads' tiles of one place,
    // the long ones first; the group's heads innermost
    int by_tile, inner;           // inner: how many of the inner kind there are
    int run;                      // consecutive pieces of work an XCD takes at a time
    int total;                    // workgroups that have work (the grid is rounded up to whole rounds of the 8 XCDs)
    float scale, sc2;             // sc2 = scale * log2(e)
};

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Workgroups are dealt to the 8 XCDs in turn.  Neighbours in the work (same keys, other head of the group; next tile) should
// share an L2, so an XCD takes runs of `run` consecutive pieces of work.
__device__ __forceinline__ int xcd_order(int block, int total, int run) {
    const int slot = block >> 3, r = uniform(slot / run);
    const int id = (r * 8 + (block & 7)) * run + slot - r * run;
    return id < total ? id : -1;
}

// BYTES a lane from a buffer (voff: the lane's byte offset; past the end reads as 0) to dst + BYTES * lane in LDS, without waiting:
// tile_ready() does.  (The compiler waits for these in front of transpose reads, which it takes for readers of what is being
// written; written in assembly, which it does not wait for, they were no faster.)
template <int BYTES> __device__ __forceinline__ void load_to_lds(const void* base, unsigned bytes, unsigned voff, void* dst) {
#if defined(__HIP_DEVICE_COMPILE__)       // the host's pass does not know the 16-byte form
    typedef __attribute__((address_space(3))) void* lds_ptr;
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, 0x00020000);
    if constexpr (BYTES == 16) __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr)(uintptr_t)dst, 16, voff, 0, 0, 0);
    else __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr)(uintptr_t)dst, 4, voff, 0, 0, 0);
#endif
}
__device__ __forceinline__ void loads_done() { __builtin_amdgcn_s_waitcnt(0x0f70); }     // vmcnt(0), in a form the compiler counts

// Rows [row0, row0 + ROWS) of a strided matrix into an image, asynchronously and without passing through registers; rows outside
// [0, hi) and columns >= dh are zero, but for rows that share memory (sn < dh: a gradient broadcast over the tokens comes with
// sn = 0): what lies behind their last row are other rows' elements, and a reader masks it.  (Zeros there too, by a branch for the
// last tile of such rows: 5 % of the backward at 64 wide heads.)  The bounds are the buffer descriptor's (what lies outside reads as
// zero), and the descriptor is moved to every tile's first row, so offsets in it stay small however long the sequence is.
// The data is there after the next tile_ready().
template <typename T, int DP, int ROWS, int NT> struct Stager {
    using C = WCfg<T, DP>;
    static constexpr int LOADS = ROWS * C::CPR / 64, CH = (LOADS + NT / 64 - 1) / (NT / 64);    // of the workgroup, of a wave
    static_assert(LOADS * 64 == ROWS * C::CPR, "a tile is a whole number of loads");
    unsigned off[CH];
    __device__ __forceinline__ void init(long sn, int dh) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int idx = threadIdx.x + c * NT;
            const int row = idx / C::CPR, d = ((idx % C::CPR) ^ C::swz(row)) * C::EPC;
            off[c] = d < dh ? (unsigned)(row * (int)sn + d) * (unsigned)sizeof(T) : 0x80000000u;
        }
    }
    __device__ __forceinline__ void load(const T* g, long sn, int row0, int hi, int dh, T* lds, int wave) const {
        const int n = min(hi - row0, ROWS);
        const unsigned bytes = n > 0 ? (unsigned)((n - 1) * (int)sn + dh) * (unsigned)sizeof(T) : 0u;
#pragma unroll
        for (int c = 0; c < CH; ++c)
            if (LOADS % (NT / 64) == 0 || c * (NT / 64) + wave < LOADS)
                load_to_lds<16>(g + (long)row0 * sn, bytes, off[c], lds + (c * NT + 64 * wave) * C::EPC);
    }
};
__device__ __forceinline__ void tile_ready() {
    asm volatile("" ::: "memory");
    loads_done();                                        // this wave's asynchronous loads; the barrier: everyone's
    __syncthreads();
}
// ROWS floats of the rows' statistics, the same way (by one wave)
template <int ROWS> __device__ __forceinline__ void load_stat(const float* g, int row0, int hi, float* lds, int lane) {
    static_assert(ROWS == 32 || ROWS % 64 == 0, "whole waves of rows, or half of one");
#pragma unroll
    for (int r = 0; r < ROWS; r += 64) {
        const int n = min(hi - row0 - r, ROWS - r);
        if (ROWS != 32 || lane < 32) load_to_lds<4>(g + row0 + r, n > 0 ? 4u * n : 0u, 4u * lane, lds + r);
    }
}

// the other half-wave's value joined in: every lane gets f of lanes l and l ^ 32
__device__ __forceinline__ float half_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
    return fmaxf(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1]));
}
__device__ __forceinline__ float half_sum(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
    return __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
}

// this wave's 32 rows of a strided matrix as fragments (rows outside [0, hi) are zero).  Loads without a branch, so that all are
// on their way together: a lane with nothing to read reads the first element and drops it.
template <typename T, int KD>
__device__ __forceinline__ void own_rows(Frag<T> (&f)[KD], const T* g, long sn, int row, int hi, int dh, int lane) {
#pragma unroll
    for (int kk = 0; kk < KD; ++kk) {
        const int d = 16 * kk + 8 * (lane >> 5);
        frag_load(f[kk], g + (row < hi && d < dh ? (long)row * sn + d : 0));
    }
#pragma unroll
    for (int kk = 0; kk < KD; ++kk)
        if (!(row < hi && 16 * kk + 8 * (lane >> 5) < dh)) frag_zero(f[kk]);
}

// X^T[d][row] (a lane owns a row) times `mul` -> rows [row0, row0 + 32) of [.][dh] with row stride ldg, turned in LDS so
// that the stores are whole chunks; rows >= hi are not written.  Only this wave's part of LDS is used.  REST: what the
// rounding to T leaves over, rounded to T.
template <typename T, int DP, bool REST = false>
__device__ __forceinline__ void put_rows(const f32x16 (&x)[DP / 32], float mul, bool zero, T* lds, T* g, long ldg, int row0, int hi, int dh,
                                         int lane) {
    using C = WCfg<T, DP>;
    typedef __attribute__((ext_vector_type(4))) T T4;
#pragma unroll
    for (int t = 0; t < DP / 32; ++t)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            T4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float y = zero ? 0.f : x[t][4 * q + e] * mul;
                if (REST) y -= (float)(T)y;
                v[e] = (T)y;
            }
            *reinterpret_cast<T4*>(lds + (lane & 31) * C::LD + 32 * t + 8 * q + 4 * (lane >> 5)) = v;
        }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    for (int idx = lane; idx < 32 * C::CPR; idx += 64) {
        const int r = idx / C::CPR, d = (idx % C::CPR) * C::EPC;
        if (row0 + r < hi && d < dh)
            *reinterpret_cast<u32x4*>(g + (long)(row0 + r) * ldg + d) = *reinterpret_cast<const u32x4*>(lds + r * C::LD + d);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

// The key tiles of BK that queries [i0, i1) can see: [0, n1) and then t0, t0 + 1, ... ; n = how many in all.
struct KeyTiles { int n1, t0, n; };
__device__ __forceinline__ KeyTiles key_tiles(const WindowParams& p, int i0, int i1, int len, int BK) {
    KeyTiles r = {0, 0, 0};
    if (i0 >= len) return r;
    int a = 0, e = len;
    if (p.causal) e = min(e, i1);
    int s = 0;                                           // one past the last sink that can be seen
    if (p.w >= 0) {
        a = max(0, i0 - p.w);
        s = min(p.S, e);
        e = (int)min((long)e, (long)i1 + p.w);
    }
    r.t0 = a / BK;
    const int t1 = (e + BK - 1) / BK, ts = (s + BK - 1) / BK;
    r.n1 = min(ts, r.t0);
    r.n = r.n1 + max(t1, ts) - r.t0;                     // sinks past the window's end follow its tiles
    return r;
}
__device__ __forceinline__ int key_tile(const KeyTiles& t, int it) { return it < t.n1 ? it : t.t0 + it - t.n1; }

// Which keys query i sees: j - lo <= span (unsigned), or j < s.
struct RowRange { int lo; unsigned span; int s; };
__device__ __forceinline__ RowRange row_range(const WindowParams& p, int i, int len) {
    RowRange r = {1 << 30, 0u, 0};
    if (i >= len) return r;
    const int e = p.causal ? i : len - 1;
    if (p.w < 0) { r.lo = 0; r.span = (unsigned)e; return r; }
    r.lo = i - p.w;                                      // p.w < N: no overflow
    r.span = (unsigned)(min(e, i + p.w) - r.lo);
    r.s = min(p.S, e + 1);
    return r;
}
constexpr int ALONE = (1 << 30) + 1;                     // RowRange::lo of such a row in the backward, past every key
__device__ __forceinline__ bool sees_itself_alone(const RowRange& r) {      // (a row within the length always sees itself)
    const int lo = max(r.lo, 0), hi = r.lo + (int)r.span;
    return lo == hi && min(r.s, lo) == 0 && r.s <= hi + 1;         // no sink before or behind its window
}
// What a wave's queries [i, i + BQ) see of keys [j0, j0 + BK): NOTHING, ALL, or which of its edges the test has to look at
enum { NOTHING = 0, ALL = 1, EDGE_HI = 2, EDGE_LO = 4, EDGE_ANY = 8 };
__device__ __forceinline__ int tile_kind(const WindowParams& p, int i, int BQ, int j0, int BK, int len) {
    if (i >= len) return NOTHING;
    const int j1 = j0 + BK - 1, i1 = i + BQ - 1;
    if (p.causal && j0 > i1) return NOTHING;
    const bool in = p.w < 0 || (j1 >= i - p.w && j0 <= i1 + p.w);
    if (!in && j0 >= p.S) return NOTHING;
    const bool hi = j1 >= len || (p.causal && j1 > i) || (p.w >= 0 && j1 > i + p.w), lo = p.w >= 0 && j0 < i1 - p.w;
    if (j1 < p.S && j1 < len && (!p.causal || j1 <= i)) return ALL;
    if (j0 < p.S && (hi || lo)) return EDGE_ANY;
    return hi ? (lo ? EDGE_ANY : EDGE_HI) : (lo ? EDGE_LO : ALL);
}
// scores of keys j0 .. that query (rr) does not see become -inf (S^T: register e of sub-tile u is key 32 u + 8 (e >> 2) + 4
// (lane >> 5) + (e & 3))
template <int NS>
__device__ __forceinline__ void hide(f32x16 (&s)[NS], int kind, const RowRange& rr, int j0, int lane) {
    const int lo = rr.lo - j0 - 4 * (lane >> 5), hi = lo + (int)rr.span, sk = rr.s - j0 - 4 * (lane >> 5);
#define VITK_HIDE(COND)                                                      \
    _Pragma("unroll") for (int u = 0; u < NS; ++u)                           \
    _Pragma("unroll") for (int e = 0; e < 16; ++e) {                         \
        const int c = 32 * u + 8 * (e >> 2) + (e & 3);                       \
        s[u][e] = (COND) ? s[u][e] : -INFINITY;                              \
    }
    if (kind == EDGE_HI) {
        VITK_HIDE(c <= hi)
    } else if (kind == EDGE_LO) {
        VITK_HIDE(c >= lo)
    } else {
        VITK_HIDE((unsigned)(c - lo) <= rr.span || c < sk)
    }
#undef VITK_HIDE
}

// Accumulators of the wave that had the other half of the keys (or queries), through LDS: at [register][lane].  Two barriers
// around the pair: put by one, added by the other.
template <int ND> __device__ __forceinline__ void half_put(float* x, const f32x16 (&a)[ND], int lane) {
#pragma unroll
    for (int t = 0; t < ND; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) x[(16 * t + e) * 64 + lane] = a[t][e];
}
template <int ND> __device__ __forceinline__ void half_add(const float* x, f32x16 (&a)[ND], float mine, float other, int lane) {
#pragma unroll
    for (int t = 0; t < ND; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) a[t][e] = a[t][e] * mine + x[(16 * t + e) * 64 + lane] * other;
}

// ---------------------------------------------------------------------------------------------------------- forward
// A wave owns 32 queries; KS = 2: two waves share them, each with one half of every tile of keys.  HW: head width in steps of 16.
// Tiles come by asynchronous loads into one of two images while the other is used, one barrier a tile.  Bound by the matrix
// unit and the softmax's vector work in turn (32 exponentials, maxima, sums and conversions of them beside 32 MFMA a wave and
// tile of 64 keys of 128): two waves a SIMD cover each other's, and no part taken out by itself gives more than 15 %.
// bf16, heads of 128: 8192 tokens x 16 heads, causal, 287 us = 960 TFLOP/s of visible pairs; 16384 tokens with a causal window
// of 1024 174 to 187 us by machine = 720 to 770, a ninth of whose pairs are the window's and the diagonal's edges and are thrown
// away (launches one after another; a profiler, which parts them, has 200 to 215).  fp32: 4 x 1001 x 16 heads of 80 195 us = 105
// TFLOP/s of 154; 2 x 2048 x 16 of 128, causal, 357 us = 96.
template <typename T, int HW, int NW, int KS, int BK, int WPE, bool FINE>
__global__ __launch_bounds__(64 * NW, WPE) void window_fwd_kernel(const WindowParams p) {
    constexpr int DP = (HW + 31) / 32 * 32;              // the width of the images
    using C = WCfg<T, DP>;
    constexpr int NT = 64 * NW, RG = NW / KS, NS = BK / 32 / KS, KD = HW / 16, ND = DP / 32, TILE = BK * DP;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    T* lds = reinterpret_cast<T*>(smem);                 // two buffers of (K tile, V tile)
    const int id = xcd_order((int)blockIdx.x, p.total, p.run);
    if (id < 0) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r1 = uniform(id / p.G), g = id - r1 * p.G;
    const int major = uniform(r1 / p.inner), minor = r1 - major * p.inner;
    const int bh = p.by_tile ? minor : major, tq = p.by_tile ? major : minor;
    const int b = uniform(bh / p.Hk), hk = bh - b * p.Hk, h = hk * p.G + g;
    const int part = KS == 1 ? 0 : uniform(wave / RG), rg = wave - part * RG;
    const int i0 = 32 * RG * (p.by_tile ? p.tiles - 1 - tq : tq), iw = i0 + 32 * rg;
    const int len = p.lengths ? uniform(max(0, min(p.lengths[b], p.N))) : p.N;
    const int i = iw + (lane & 31);

    const T* K = static_cast<const T*>(p.k.p) + (long)b * p.k.sb + (long)hk * p.k.sh;
    const T* V = static_cast<const T*>(p.v.p) + (long)b * p.v.sb + (long)hk * p.v.sh;
    Frag<T> qf[KD];
    own_rows<T, KD>(qf, static_cast<const T*>(p.q.p) + (long)b * p.q.sb + (long)h * p.q.sh, p.q.sn, i, len, p.dh, lane);

    const KeyTiles kt = key_tiles(p, i0, i0 + 32 * RG, len, BK);
    const RowRange rr = row_range(p, i, len);
    f32x16 o[ND];
    float m;                                             // running maximum, log2 domain
    float ls[4];                                         // the sum of this lane's keys, in four chains

    loads_done();                                        // nothing but tiles is in flight in the loop
    Stager<T, DP, BK, NT> sk, sv;
    sk.init(p.k.sn, p.dh);
    sv.init(p.v.sn, p.dh);
    auto walk = [&](auto careful) {
        m = -INFINITY;
#pragma unroll
        for (int e = 0; e < 4; ++e) ls[e] = 0.f;
#pragma unroll
        for (int t = 0; t < ND; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[t][e] = 0.f;
        if (kt.n > 0) {
            const int j0 = BK * key_tile(kt, 0);
            sk.load(K, p.k.sn, j0, len, p.dh, lds, wave);
            sv.load(V, p.v.sn, j0, len, p.dh, lds + TILE, wave);
        }
        for (int it = 0; it < kt.n; ++it) {
            const T* Ks = lds + (it & 1) * 2 * TILE + part * (32 * NS * DP);
            const T* Vs = Ks + TILE;
            tile_ready();                                    // and the other buffer's readers are done
            if (it + 1 < kt.n) {
                const int j1 = BK * key_tile(kt, it + 1);
                T* nx = lds + ((it + 1) & 1) * 2 * TILE;
                sk.load(K, p.k.sn, j1, len, p.dh, nx, wave);
                sv.load(V, p.v.sn, j1, len, p.dh, nx + TILE, wave);
            }
            const int j0 = BK * key_tile(kt, it) + 32 * NS * part;
            const int kind = tile_kind(p, iw, 32, j0, 32 * NS, len);         // the same for the whole wave
            if (kind) {
                f32x16 s[NS];
                float mt = -INFINITY;
#pragma unroll
                for (int u = 0; u < NS; ++u) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[u][e] = 0.f;
#pragma unroll
                    for (int kk = 0; kk < KD; ++kk) {
                        Frag<T> a;
                        row_frag32<DP>(a, Ks, 32 * u, kk, lane);
                        s[u] = mma32(a, qf[kk], s[u]);
                    }
                }
                if (kind != ALL) hide(s, kind, rr, j0, lane);
#pragma unroll
                for (int u = 0; u < NS; ++u)
#pragma unroll
                    for (int e = 0; e < 16; ++e) mt = fmaxf(mt, s[u][e]);
                mt = half_max(mt) * p.sc2;
                // the reference point only has to keep exp2 in range: it moves when a row's maximum has grown by 2^8
                if (__any(mt > m + 8.f)) {
                    const float mn = fmaxf(m, mt);
                    const float al = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
                    m = mn;
#pragma unroll
                    for (int e = 0; e < 4; ++e) ls[e] *= al;
#pragma unroll
                    for (int t = 0; t < ND; ++t)
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[t][e] *= al;
                }
                const float mr = m == -INFINITY ? 0.f : m;
                if (__any(fabsf(mr) > 16777216.f)) {         // out here the product's rounding, which m has and the fma has not,
#pragma unroll                                           // would be an exponent of its own
                    for (int u = 0; u < NS; ++u)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            float x = s[u][e] * p.sc2;
                            asm("" : "+v"(x));               // two roundings: not to be contracted
                            s[u][e] = x - mr;
                        }
                } else {
#pragma unroll
                    for (int u = 0; u < NS; ++u)
#pragma unroll
                        for (int e = 0; e < 16; ++e) s[u][e] = fmaf(s[u][e], p.sc2, -mr);
                }
                if constexpr (decltype(careful)::value) {                // no visible key's p is 0
#pragma unroll
                    for (int u = 0; u < NS; ++u)
#pragma unroll
                        for (int e = 0; e < 16; ++e) s[u][e] = s[u][e] < -120.f && s[u][e] > -INFINITY ? -120.f : s[u][e];
                }
#pragma unroll
                for (int u = 0; u < NS; ++u)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        s[u][e] = __builtin_amdgcn_exp2f(s[u][e]);
                        ls[e & 3] += s[u][e];
                    }
                if constexpr (decltype(careful)::value) {
#pragma unroll
                    for (int t = 0; t < ND; ++t) {
#pragma unroll
                        for (int part = 0; part < 3; ++part) {           // the finite values, then where +inf and -inf go
                            f32x16 c = o[t];
                            if (part) {
#pragma unroll
                                for (int e = 0; e < 16; ++e) c[e] = 0.f;
                            }
#pragma unroll
                            for (int u = 0; u < NS; ++u)
#pragma unroll
                                for (int ks = 0; ks < 2; ++ks) {
                                    Frag<T> a, pf, rest;
                                    asm volatile("" ::: "memory");       // one product's operands in registers at a time
                                    __builtin_amdgcn_sched_barrier(0);
                                    int l2 = lane;
                                    asm volatile("" : "+v"(l2));
                                    col_frag32<DP>(a, Vs, 32 * u + 16 * ks, 32 * t, l2);
                                    value_part(a, part);
                                    acc_frag(pf, s[u], ks);
                                    if constexpr (FINE) {
                                        rest_frag(rest, pf, s[u], ks);
                                        if (!part) c = mma32(a, rest, c);
                                    }
                                    if (part) {
#pragma unroll
                                        for (int e = 0; e < 8; ++e) frag_set_f(pf, e, s[u][8 * ks + e] > 0.f ? 1.f : 0.f);
                                    }
                                    c = mma32(a, pf, c);
                                }
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                if (!part) o[t][e] = c[e];
                                else o[t][e] += c[e] > 0.f ? (part == 1 ? INFINITY : -INFINITY) : 0.f;
                            }
                        }
                    }
                } else
#pragma unroll
                for (int u = 0; u < NS; ++u)
#pragma unroll
                    for (int ks = 0; ks < 2; ++ks) {
                        Frag<T> pf, rest;
                        acc_frag(pf, s[u], ks);
                        if constexpr (FINE) rest_frag(rest, pf, s[u], ks);
#pragma unroll
                        for (int t = 0; t < ND; ++t) {
                            Frag<T> a;
                            col_frag32<DP>(a, Vs, 32 * u + 16 * ks, 32 * t, lane);
                            o[t] = mma32(a, pf, o[t]);
                            if constexpr (FINE) o[t] = mma32(a, rest, o[t]);
                        }
                    }
            }
        }
    };
    walk(std::false_type{});
    float l = half_sum((ls[0] + ls[1]) + (ls[2] + ls[3]));
    // A non-finite V of a key that only some queries of a tile see has reached the others as 0 * V.  Where a result is not finite,
    // the workgroup walks again and multiplies the finite values, and 0 and 1 for the infinities, apart.  (FINE: p and its
    // remainder can be of two signs, and infinity times both is no number.  V rows that share memory: what lies behind the last
    // one is hidden too.)
    __shared__ int again[NW];
    {
        float bad = 0.f;
#pragma unroll
        for (int t = 0; t < ND; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) bad += o[t][e] * 0.f;
        const bool redo = __any(i < len && bad != 0.f && l == l);        // (a NaN is unequal; a NaN sum is the row's own)
        if (lane == 0) again[wave] = redo;
    }
    __syncthreads();                                     // everyone is done with the tiles
    int redo = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) redo |= again[w];
    if (__builtin_expect((FINE || p.w >= 0 || p.causal || p.v.sn < p.dh) && uniform(redo), 0)) {
        walk(std::true_type{});
        l = half_sum((ls[0] + ls[1]) + (ls[2] + ls[3]));
        __syncthreads();
    }
    if constexpr (KS == 2) {
        float* x = reinterpret_cast<float*>(smem) + rg * (16 * ND + 2) * 64;
        if (part) {
            half_put(x, o, lane);
            x[16 * ND * 64 + lane] = m;
            x[16 * ND * 64 + 64 + lane] = l;
        }
        __syncthreads();
        if (!part) {
            const float m1 = x[16 * ND * 64 + lane], l1 = x[16 * ND * 64 + 64 + lane], mn = fmaxf(m, m1);
            const float f0 = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn), f1 = m1 == mn ? 1.f : __builtin_amdgcn_exp2f(m1 - mn);
            half_add(x, o, f0, f1, lane);
            l = l * f0 + l1 * f1;
            m = mn;
        }
        __syncthreads();
        if (part) return;
    }
    const bool none = i >= len || (m == -INFINITY && l == 0.f);      // nothing visible (a NaN sum stays a NaN)
    if (p.lse && lane < 32 && i < p.N) p.lse[((long)b * p.Hq + h) * p.N + i] = none ? INFINITY : m + __log2f(l);
    const long at = ((long)b * p.N * p.Hq + h) * p.dh, ldg = (long)p.Hq * p.dh;
    T* mine = lds + rg * 32 * C::LD;
    put_rows<T, DP>(o, 1.f / l, none, mine, static_cast<T*>(p.out) + at, ldg, iw, p.N, p.dh, lane);
    if (sizeof(T) == 2 && p.o_lo) put_rows<T, DP, true>(o, 1.f / l, none, mine, static_cast<T*>(p.o_lo) + at, ldg, iw, p.N, p.dh, lane);
}

// The backward makes P again as exp2(score - lse), and lse's rounding is an error of its whole row: 2^-16 of P at most up to an
// |lse| of FAR, but 2^-4 at a million, and past FAR_ROUNDED, where the forward rounds the products, a power of two of its own.
// Where one of 32 rows is out there (a diverging model's), all of them take their scores minus lse for scores, with a log-sum of
// 0, and have P's sum made again beside dq to divide by.  That is a second copy of the loops, which a workgroup takes if it
// meets such rows: a test within the loops cost 4 to 8 % of the backward, this 0 to 2.
constexpr float FAR = 512.f, FAR_ROUNDED = 16777216.f;
__device__ __forceinline__ bool beyond(float lse, float limit) { return !(fabsf(lse) <= limit); }
__device__ __forceinline__ float far_exponent(float s, float sc2, float lse, bool rounded) {
    float x = s * sc2;
    asm("" : "+v"(x));                                   // two roundings: not to be contracted
    return rounded ? x - lse : fmaf(s, sc2, -lse);
}

// ------------------------------------------------------------------------------------- backward: dq (and D for the other)
// The forward's walk with three products (S, dP, dS K); 275 us = 730 TFLOP/s at the forward's windowed size.
template <typename T, int HW, int NW, int KS, int BK, int WPE, bool FINE>
__global__ __launch_bounds__(64 * NW, WPE) void window_dq_kernel(const WindowParams p) {
    constexpr int DP = (HW + 31) / 32 * 32;              // the width of the images
    using C = WCfg<T, DP>;
    constexpr int NT = 64 * NW, RG = NW / KS, NS = BK / 32 / KS, KD = HW / 16, ND = DP / 32, TILE = BK * DP;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    T* lds = reinterpret_cast<T*>(smem);
    const int id = xcd_order((int)blockIdx.x, p.total, p.run);
    if (id < 0) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r1 = uniform(id / p.G), g = id - r1 * p.G;
    const int major = uniform(r1 / p.inner), minor = r1 - major * p.inner;
    const int bh = p.by_tile ? minor : major, tq = p.by_tile ? major : minor;
    const int b = uniform(bh / p.Hk), hk = bh - b * p.Hk, h = hk * p.G + g;
    const int part = KS == 1 ? 0 : uniform(wave / RG), rg = wave - part * RG;
    const int i0 = 32 * RG * (p.by_tile ? p.tiles - 1 - tq : tq), iw = i0 + 32 * rg;
    const int len = p.lengths ? uniform(max(0, min(p.lengths[b], p.N))) : p.N;
    const int i = iw + (lane & 31);

    const T* K = static_cast<const T*>(p.k.p) + (long)b * p.k.sb + (long)hk * p.k.sh;
    const T* V = static_cast<const T*>(p.v.p) + (long)b * p.v.sb + (long)hk * p.v.sh;
    Frag<T> qf[KD], df[KD];
    own_rows<T, KD>(qf, static_cast<const T*>(p.q.p) + (long)b * p.q.sb + (long)h * p.q.sh, p.q.sn, i, len, p.dh, lane);
    own_rows<T, KD>(df, static_cast<const T*>(p.dout.p) + (long)b * p.dout.sb + (long)h * p.dout.sh, p.dout.sn, i, len, p.dh, lane);
    // a row that sees nothing but its own key has dS = 0, and exactly so: D is what the products make of do . v, dP's own bits
    RowRange rr = row_range(p, i, len);
    if (i < len && sees_itself_alone(rr)) rr = RowRange{ALONE, 0u, 0};
    float delta = 0.f, lse = INFINITY;
    {
        // with o as it was rounded, D's error is the same for all of a row's keys and reaches dq and dk whole: as much again as
        // the rounding of dS where a row sees few keys
        const long row = ((long)b * p.N * p.Hq + h) * p.dh;
        Frag<T> of[KD], lo[KD];
        own_rows<T, KD>(of, static_cast<const T*>(p.o) + row, (long)p.Hq * p.dh, i, len, p.dh, lane);
        if (sizeof(T) == 2 && p.o_lo) own_rows<T, KD>(lo, static_cast<const T*>(p.o_lo) + row, (long)p.Hq * p.dh, i, len, p.dh, lane);
#pragma unroll
        for (int kk = 0; kk < KD; ++kk)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = frag_get_f(of[kk], e), d = frag_get_f(df[kk], e);
                delta += (sizeof(T) == 2 && p.o_lo ? x + frag_get_f(lo[kk], e) : x) * d;
            }
        delta = half_sum(delta);
        const long at = ((long)b * p.Hq + h) * p.N + i;
        if (i < len) lse = p.lse[at];
        if (!part && rr.lo != ALONE && lane < 32 && i < p.N) p.delta[at] = delta;
    }
    bool any_far = false;                                // the same for the whole workgroup
#pragma unroll
    for (int r = 0; r < 32 * RG; r += 64) {
        const int row = i0 + r + lane;
        any_far |= __any(row < len && beyond(p.lse[((long)b * p.Hq + h) * p.N + min(row, p.N - 1)], FAR)) != 0;
    }
    const bool far = __any(i < len && beyond(lse, FAR));
    float total = 0.f;                                   // far: the sum of P over this lane's keys
    if (!part && lane == 0 && iw < len) p.far[((long)b * p.Hq + h) * ((p.N + 31) / 32) + iw / 32] = far;
    const KeyTiles kt = key_tiles(p, i0, i0 + 32 * RG, len, BK);
    f32x16 dq[ND];
#pragma unroll
    for (int t = 0; t < ND; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) dq[t][e] = 0.f;

    loads_done();                                        // nothing but tiles is in flight in the loop
    Stager<T, DP, BK, NT> sk, sv;
    sk.init(p.k.sn, p.dh);
    sv.init(p.v.sn, p.dh);
    if (kt.n > 0) {
        const int j0 = BK * key_tile(kt, 0);
        sk.load(K, p.k.sn, j0, len, p.dh, lds, wave);
        sv.load(V, p.v.sn, j0, len, p.dh, lds + TILE, wave);
    }
    auto walk = [&](auto fars) {
        constexpr bool FARS = decltype(fars)::value;
        for (int it = 0; it < kt.n; ++it) {
            const T* Ks = lds + (it & 1) * 2 * TILE + part * (32 * NS * DP);
            const T* Vs = Ks + TILE;
            tile_ready();
            if (it + 1 < kt.n) {
                const int j1 = BK * key_tile(kt, it + 1);
                T* nx = lds + ((it + 1) & 1) * 2 * TILE;
                sk.load(K, p.k.sn, j1, len, p.dh, nx, wave);
                sv.load(V, p.v.sn, j1, len, p.dh, nx + TILE, wave);
            }
            const int j0 = BK * key_tile(kt, it) + 32 * NS * part;
            const int kind = tile_kind(p, iw, 32, j0, 32 * NS, len);
            if (kind) {
#pragma unroll
                for (int u = 0; u < NS; ++u) {
                    f32x16 s, dp;
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[e] = dp[e] = 0.f;
#pragma unroll
                    for (int kk = 0; kk < KD; ++kk) {
                        Frag<T> a;
                        row_frag32<DP>(a, Ks, 32 * u, kk, lane);
                        s = mma32(a, qf[kk], s);
                        row_frag32<DP>(a, Vs, 32 * u, kk, lane);
                        dp = mma32(a, df[kk], dp);
                    }
                    if (j0 + 32 * u == iw && __any(rr.lo == ALONE)) {
                        float own = 0.f;
#pragma unroll
                        for (int e = 0; e < 16; ++e) own = 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3) == (lane & 31) ? dp[e] : own;
                        own = half_sum(own);
                        if (rr.lo == ALONE && lane < 32) p.delta[((long)b * p.Hq + h) * p.N + i] = own;
                    }
                    float ref = lse;
                    if constexpr (FARS) {
                        if (far) {
                            const bool rounded = __any(i < len && beyond(lse, FAR_ROUNDED));
                            const float inv = 1.f / p.sc2;
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                const int j = j0 + 32 * u + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
                                const float y = far_exponent(s[e], p.sc2, lse, rounded);
                                const bool ok = rr.lo == ALONE ? j == i : (unsigned)(j - rr.lo) <= rr.span || j < rr.s;
                                total += ok ? __builtin_amdgcn_exp2f(y) : 0.f;
                                s[e] = y * inv;
                            }
                            ref = 0.f;
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], p.sc2, -ref)) * (dp[e] - delta);
                    if (kind != ALL) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int j = j0 + 32 * u + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
                            const bool ok = (unsigned)(j - rr.lo) <= rr.span || j < rr.s;
                            s[e] = ok ? s[e] : 0.f;
                        }
                    }
#pragma unroll
                    for (int ks = 0; ks < 2; ++ks) {
                        Frag<T> sf, rest;
                        acc_frag(sf, s, ks);
                        if constexpr (FINE) rest_frag(rest, sf, s, ks);
#pragma unroll
                        for (int t = 0; t < ND; ++t) {
                            Frag<T> a;
                            col_frag32<DP>(a, Ks, 32 * u + 16 * ks, 32 * t, lane);
                            dq[t] = mma32(a, sf, dq[t]);
                            if constexpr (FINE) dq[t] = mma32(a, rest, dq[t]);
                        }
                    }
                }
            }
        }
    };
    if (__builtin_expect(!any_far, 1)) walk(std::false_type{});
    else walk(std::true_type{});
    __syncthreads();
    if constexpr (KS == 2) {
        float* x = reinterpret_cast<float*>(smem) + rg * (16 * ND + 1) * 64;
        if (part) {
            half_put(x, dq, lane);
            x[16 * ND * 64 + lane] = total;
        }
        __syncthreads();
        if (!part) {
            half_add(x, dq, 1.f, 1.f, lane);
            total += x[16 * ND * 64 + lane];
        }
        __syncthreads();
        if (part) return;
    }
    float mul = p.scale;
    if (far) {
        total = half_sum(total);
        if (total == 0.f) total = 1.f;                   // every score is -inf: the row is zero, and stays it
        mul /= total;
        if (lane < 32 && i < len) p.shift[((long)b * p.Hq + h) * p.N + i] = -__log2f(total);
    }
    put_rows<T, DP>(dq, mul, i >= len, lds + rg * 32 * C::LD, static_cast<T*>(p.out) + ((long)b * p.N * p.Hq + h) * p.dh,
                    (long)p.Hq * p.dh, iw, p.N, p.dh, lane);
}

// --------------------------------------------------------------------------------------------- backward: dk and dv
// A wave owns 32 keys (a lane one key, scores S[query][key]); the workgroup walks the query tiles that can see its keys, for
// every head of the group.  KS waves share 32 keys, each with its own part of every query tile.  SINK: the 32 keys of a sinks'
// tile and a share of ALL the query tiles, each wave's sums out in fp32 (window_sink_sum_kernel adds the shares in order).
// Four products (S, dP, P dO, dS Q) on the same two operands: 320 us = 830 TFLOP/s at the forward's windowed size.  fp32 is one
// wave a SIMD from 80 wide heads on (194 + 128 registers): 4 x 1001 x 16 of 80 672 us for the whole backward.
template <typename T, int HW, int NW, int KS, int BQ, bool SINK, bool VLDS, int WPE, bool FINE>
__global__ __launch_bounds__(64 * NW, WPE) void window_dkv_kernel(const WindowParams p) {
    constexpr int DP = (HW + 31) / 32 * 32;              // the width of the images
    using C = WCfg<T, DP>;
    constexpr int NT = 64 * NW, RG = NW / KS, NS = BQ / 32 / KS, KD = HW / 16, ND = DP / 32, TILE = BQ * DP;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    T* lds = reinterpret_cast<T*>(smem);                 // two buffers of (Q tile, dO tile), then of BQ (lse, D) each
    float* stat = reinterpret_cast<float*>(lds + 4 * TILE);
    // tiles with sinks in an ordinary launch take longest and go first, one to each XCD in turn
    const int first = p.heavy * p.B * p.Hk, round = (first + 7) / 8 * 8;
    int id, chunk = 0, bh, tk;
    if ((int)blockIdx.x < round) {
        id = (int)blockIdx.x < first ? (int)blockIdx.x : -1;
        bh = uniform((int)blockIdx.x / max(p.heavy, 1));
        tk = (int)blockIdx.x - bh * p.heavy;
    } else {
        id = xcd_order((int)blockIdx.x - round, p.total, p.run);
        int r1 = max(id, 0);
        if (SINK) {
            chunk = r1;
            r1 = uniform(r1 / p.chunks);
            chunk -= r1 * p.chunks;
        }
        const int major = uniform(r1 / p.inner), minor = r1 - major * p.inner;
        bh = p.by_tile ? minor : major;
        tk = p.by_tile ? (p.causal ? p.heavy + major : p.tiles - 1 - major) : p.heavy + minor;
    }
    if (id < 0) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = uniform(bh / p.Hk), hk = bh - b * p.Hk;
    const int part = KS == 1 ? 0 : uniform(wave / RG), rg = wave - part * RG;
    const int j0 = p.key0 + 32 * RG * tk, jw = j0 + 32 * rg, j = jw + (lane & 31);
    const int len = p.lengths ? uniform(max(0, min(p.lengths[b], p.N))) : p.N;

    Frag<T> kf[KD], vf[VLDS ? 1 : KD];
    T* Vs = reinterpret_cast<T*>(stat + 4 * BQ);         // VLDS: the workgroup's V rows stay in LDS
    own_rows<T, KD>(kf, static_cast<const T*>(p.k.p) + (long)b * p.k.sb + (long)hk * p.k.sh, p.k.sn, j, len, p.dh, lane);
    const T* V = static_cast<const T*>(p.v.p) + (long)b * p.v.sb + (long)hk * p.v.sh;
    if constexpr (!VLDS) own_rows<T, KD>(vf, V, p.v.sn, j, len, p.dh, lane);

    // queries that see key j: i - ilo <= span (unsigned); none for a key past the end
    int ilo = 1 << 30;
    unsigned span = 0;
    if (j < len) {
        const bool all = p.w < 0 || j < p.S;
        ilo = p.causal ? j : (all ? 0 : max(0, j - p.w));
        span = (unsigned)((all ? len - 1 : min(len - 1, j + p.w)) - ilo);
    }
    // query tiles [ta, ta + nt) of each of the group's heads
    int ta = 0, nt = 0;
    if (j0 < len) {
        int a = p.causal ? j0 : 0, e = len;
        if (p.w >= 0 && j0 >= p.S) {                     // (the sinks' tiles are seen from everywhere)
            a = max(a, j0 - p.w);
            e = (int)min((long)e, (long)j0 + 32 * RG + p.w);
        }
        ta = a / BQ;
        nt = (e + BQ - 1) / BQ - ta;
    }
    const int items = nt * p.G;
    const int it0 = SINK ? min(items, chunk * p.per_chunk) : 0, it1 = SINK ? min(items, it0 + p.per_chunk) : items;

    f32x16 dk[ND], dv[ND];
#pragma unroll
    for (int t = 0; t < ND; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) dk[t][e] = dv[t][e] = 0.f;

    loads_done();
    if constexpr (VLDS) {
        Stager<T, DP, 32 * RG, NT> sv;
        sv.init(p.v.sn, p.dh);
        sv.load(V, p.v.sn, j0, len, p.dh, Vs, wave);
    }
    Stager<T, DP, BQ, NT> sq, sd;
    sq.init(p.q.sn, p.dh);
    sd.init(p.dout.sn, p.dh);
    auto fetch = [&](int it) {
        const int gi = uniform(it / nt), h = hk * p.G + gi, i0 = BQ * (ta + it - gi * nt);
        T* nx = lds + (it & 1) * 2 * TILE;
        sq.load(static_cast<const T*>(p.q.p) + (long)b * p.q.sb + (long)h * p.q.sh, p.q.sn, i0, len, p.dh, nx, wave);
        sd.load(static_cast<const T*>(p.dout.p) + (long)b * p.dout.sb + (long)h * p.dout.sh, p.dout.sn, i0, len, p.dh, nx + TILE, wave);
        float* ns = stat + (it & 1) * 2 * BQ;
        const long at = ((long)b * p.Hq + h) * p.N;
        if (wave == 0) load_stat<BQ>(p.lse + at, i0, len, ns, lane);
        if (wave == NW - 1) load_stat<BQ>(p.delta + at, i0, len, ns + BQ, lane);
    };
    // 32 queries of a tile: scores and dP, P and dS from them, then dv and dk
    auto tile = [&](auto fars, int kind, const T* Qs, const T* Ds, const float* ls, int u, int i0, int it) {
        f32x16 s, dp;
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = dp[e] = 0.f;
#pragma unroll
        for (int kk = 0; kk < KD; ++kk) {
            Frag<T> a, v;
            row_frag32<DP>(a, Qs, 32 * u, kk, lane);
            s = mma32(a, kf[kk], s);
            row_frag32<DP>(a, Ds, 32 * u, kk, lane);
            if constexpr (VLDS) {
                row_frag32<DP>(v, Vs, 32 * rg, kk, lane);
                dp = mma32(a, v, dp);
            } else {
                dp = mma32(a, vf[kk], dp);
            }
        }
        bool far = false;
        if constexpr (decltype(fars)::value) {
            const int r0 = i0 + 32 * u;                  // (before the end, or there would be nothing to see)
            const long bh = (long)b * p.Hq + hk * p.G + uniform(it / nt);
            far = uniform(p.far[bh * ((p.N + 31) / 32) + r0 / 32]);
            if (far) {
                const float* lse = p.lse + bh * p.N;
                const bool rounded = __any(beyond(lse[min(r0 + (lane & 31), len - 1)], FAR_ROUNDED));
                const float inv = 1.f / p.sc2;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int r = min(r0 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3), len - 1);
                    asm volatile("" ::: "memory");
                    s[e] = (far_exponent(s[e], p.sc2, lse[r], rounded) + p.shift[bh * p.N + r]) * inv;
                }
            }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int row = 32 * u + 8 * q + 4 * (lane >> 5);
            asm volatile("" ::: "memory");               // one quarter's statistics in registers at a time
            f32x4 L = *reinterpret_cast<const f32x4*>(ls + row), D = *reinterpret_cast<const f32x4*>(ls + BQ + row);
            if (far) L = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float pe = __builtin_amdgcn_exp2f(fmaf(s[4 * q + e], p.sc2, -L[e]));
                dp[4 * q + e] = pe * (dp[4 * q + e] - D[e]);
                s[4 * q + e] = pe;
            }
        }
        if (kind != ALL) {                               // (no second copy of the products: it costs moves of all accumulators)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const bool ok = (unsigned)(i0 + 32 * u + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3) - ilo) <= span;
                s[e] = ok ? s[e] : 0.f;
                dp[e] = ok ? dp[e] : 0.f;
            }
        }
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            Frag<T> pf, sf, pr, sr;
            acc_frag(pf, s, ks);
            acc_frag(sf, dp, ks);
            if constexpr (FINE) {
                rest_frag(pr, pf, s, ks);
                rest_frag(sr, sf, dp, ks);
            }
#pragma unroll
            for (int t = 0; t < ND; ++t) {
                Frag<T> a;
                col_frag32<DP>(a, Ds, 32 * u + 16 * ks, 32 * t, lane);
                dv[t] = mma32(a, pf, dv[t]);
                if constexpr (FINE) dv[t] = mma32(a, pr, dv[t]);
                col_frag32<DP>(a, Qs, 32 * u + 16 * ks, 32 * t, lane);
                dk[t] = mma32(a, sf, dk[t]);
                if constexpr (FINE) dk[t] = mma32(a, sr, dk[t]);
            }
        }
    };
    if (it0 < it1) fetch(it0);
    bool any_far = false;                                // the same for the whole workgroup; read beside the first tile
    {
        const int groups = (p.N + 31) / 32, per = BQ / 32;
        for (int x = it0 * per + lane; x < it1 * per; x += 64) {
            const int gi = x / (nt * per), at = ta * per + x - gi * (nt * per);
            any_far |= 32 * at < len && p.far[((long)b * p.Hq + hk * p.G + gi) * groups + at];
        }
        any_far = __any(any_far);
    }
    auto walk = [&](auto fars) {
        for (int it = it0; it < it1; ++it) {
            const T* Qs = lds + (it & 1) * 2 * TILE + part * (32 * NS * DP);
            const T* Ds = Qs + TILE;
            const float* ls = stat + (it & 1) * 2 * BQ + 32 * NS * part;
            tile_ready();
            if (it + 1 < it1) fetch(it + 1);
            const int i0 = BQ * (ta + it - uniform(it / nt) * nt) + 32 * NS * part;
#pragma unroll
            for (int u = 0; u < NS; ++u) {
                int kind = jw < len ? tile_kind(p, i0 + 32 * u, 32, jw, 32, len) : 0;
                // queries past the end: their statistics come as zeros, so p is 1 or more there, and dO's and Q's rows may be others'
                if (kind && i0 + 32 * u + 32 > len) kind = EDGE_ANY;
                if (kind) tile(fars, kind, Qs, Ds, ls, u, i0, it);
            }
        }
    };
    if (any_far) walk(std::true_type{});
    else walk(std::false_type{});
    if (SINK) {
        float* o = p.part + ((long)id * KS + part) * 2 * DP * 32;
#pragma unroll
        for (int t = 0; t < ND; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int d = 32 * t + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
                o[d * 32 + (lane & 31)] = dk[t][e];
                o[(DP + d) * 32 + (lane & 31)] = dv[t][e];
            }
        return;
    }
    __syncthreads();
    if constexpr (KS == 2) {
        float* x = reinterpret_cast<float*>(smem) + rg * 32 * ND * 64;
        if (part) {
            half_put(x, dk, lane);
            half_put(x + 16 * ND * 64, dv, lane);
        }
        __syncthreads();
        if (!part) {
            half_add(x, dk, 1.f, 1.f, lane);
            half_add(x + 16 * ND * 64, dv, 1.f, 1.f, lane);
        }
        __syncthreads();
        if (part) return;
    }
    T* mine = lds + rg * 32 * C::LD;
    const long at = ((long)b * p.N * p.Hk + hk) * p.dh, ldg = (long)p.Hk * p.dh;
    put_rows<T, DP>(dk, p.scale, j >= len, mine, static_cast<T*>(p.dk) + at, ldg, jw, p.N, p.dh, lane);
    put_rows<T, DP>(dv, 1.f, j >= len, mine, static_cast<T*>(p.dv) + at, ldg, jw, p.N, p.dh, lane);
}

// rows of the sinks' tiles: the shares' sum in a fixed order, rounded once.  A workgroup takes 2 head elements of one (sequence,
// key head, tile), dk or dv, times 32 keys; each of its waves a quarter of the shares.
template <typename T, int DP>
__global__ __launch_bounds__(256) void window_sink_sum_kernel(const WindowParams p) {
    __shared__ float t[4][64];
    const int d0 = 2 * (blockIdx.x % (DP / 2)), which = blockIdx.x / (DP / 2) % 2;
    const int set = blockIdx.x / (DP / 2) / 2;
    const int bh = set / p.tiles, tk = set - bh * p.tiles;
    const int b = bh / p.Hk, hk = bh - b * p.Hk;
    if (d0 >= p.dh) return;
    const int lane = threadIdx.x & 63, part = threadIdx.x >> 6, per = (p.chunks + 3) / 4;
    const float* from = p.part + ((long)set * p.chunks * 2 + which) * DP * 32 + d0 * 32 + lane;
    const int c1 = min(p.chunks, (part + 1) * per);
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    int c = part * per;
    for (; c + 8 <= c1; c += 8)
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] += from[(long)(c + e) * 2 * DP * 32];
    for (; c < c1; ++c) s[0] += from[(long)c * 2 * DP * 32];
    t[part][lane] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
    __syncthreads();
    const int j = 32 * tk + (lane >> 1), at = 32 * (lane & 1) + (lane >> 1);     // two neighbours hold one key's two elements
    if (part == 0 && j < p.N) {
        const float sum = (t[0][at] + t[1][at]) + (t[2][at] + t[3][at]);
        static_cast<T*>(which ? p.dv : p.dk)[(((long)b * p.N + j) * p.Hk + hk) * p.dh + d0 + (lane & 1)] = (T)(which ? sum : sum * p.scale);
    }
}

}  // namespace vitk

using namespace vitk;

namespace {

struct Plan {                  // tiles of one call
    int dp;                    // staged head width: 32, 64, 96 or 128
    int width;                 // the width that the products over head elements take: dp, or 80 (in steps of 16)
    bool halves_q, halves_k;   // workgroups of 64 queries / keys whose rows are shared by two waves each, else of 128
    int sink_keys;             // keys that the sinks' launch takes (a multiple of 32, 0: none)
    int chunks, per_chunk;     // workgroups a sinks' tile, query tiles each of them takes
    int shares;                // partial sums that they leave
    bool fine;                 // bf16: P and dS as two bf16 each
};
constexpr long FINE = 1 << 17;
constexpr int SINK_ITEMS = 24;
constexpr int sink_waves(int bytes_of_a_row) { return bytes_of_a_row <= 128 ? 4 : 2; }       // 4 tiles of 32 rows each for them in LDS
constexpr int NARROW = 256;

// Up to how many workgroups of 128 rows there are, that workgroups of 64 with two waves a row, each with half of the other axis,
// are faster.  One of 128 takes as long as its longest row, whatever the other CUs do: few of them leave CUs, and a second
// round of them most of its CUs, waiting.  Halves read every tile for half the rows.  fp32, 16 heads x 1001 tokens of 80, forward
// and backward: one sequence 67 + 192 us against 113 + 349, three 186 + 571 against 193 + 664, four 249 + 763 against 195 +
// 673; causal, four of 1024: 143 + 436 against 148 + 436.  bf16, 16 x 1024: heads of 128, causal, 23 + 62 against 30 + 95, two
// sequences 26 + 74 against 32 + 96, three 34 + 108 against 33 + 102; of 64 three 26 + 75 against 27 + 79, four 32 + 94 against 29 + 83.
long halves_up_to(int dtype, int dp, bool uneven) { return dtype == VITK_F32 ? (uneven ? 512 : 384) : (dp <= 64 ? 384 : 256); }

Plan make_plan(int dtype, int B, int N, int Hq, int Hk, int dh, int w, int S, bool causal, bool uneven) {
    Plan pl;
    pl.dp = (dh + 31) / 32 * 32;
    pl.width = dh > 64 && dh <= 80 ? 80 : pl.dp;         // (4 x 1001 x 16 heads of 80, fp32: 195 + 672 us
                                                         // forward and backward; as 96, a sixth more steps, 209 + 730; bf16 40 + 114, 39 + 120)
    // P and dS are rounded to bf16 for their products, an error of the size of the results' own rounding as long as many share in
    // it.  In a call of few scores single ones can carry dq and dk (up to 87 tokens, window 2: 0.0021 of the norm before the
    // result's own rounding, 0.0017 in large calls): there what the rounding took is multiplied too, in the forward as well,
    // whose error dq and dk have through o . do (180 tokens x 4 heads of 64: forward 8.1 us against 7.7, backward 18.6 against
    // 17.4).
    const long keys = w < 0 ? N : (2L * w + 1 + S < N ? 2L * w + 1 + S : N);
    pl.fine = dtype == VITK_BF16 && (long)B * Hq * N * keys <= FINE;
    const long tq = (long)B * Hq * ((N + 127) / 128), tk = (long)B * Hk * ((N + 127) / 128), most = halves_up_to(dtype, pl.dp, uneven);
    pl.halves_q = pl.fine || tq <= most;
    // (causal without a window: the first keys' rows are twice the average, times the group's heads.  8 ragged sequences up to 1500
    // x 16 heads of 80 in groups of 4: the backward 198 us against 283; 2 x 8192 x 12 of 64 in groups of 3: 866 against 1013)
    pl.halves_k = pl.fine || tk <= (dtype == VITK_BF16 && causal && w < 0 ? 2 * most : most);
    // The sinks' keys are seen by all N queries, the 128 of another tile by `near` of them.  Where that is over four times more, or
    // so much that the ordinary launch would wait for the sinks' tiles, they get a launch of their own, whose workgroups share
    // the queries, and a sum; else they go first in the ordinary one (16 x 577 tokens x 12 heads, window 64: 37 us in all
    // against 33 + 14 + 7; backward of 1 x 577 x 12: 26 against 31, of 1001 tokens x 8 heads in groups of 4, causal window of
    // 100: 85 against 44, fp32 314 against 125).
    const long near = 128 + (causal ? 1L : 2L) * w;
    const bool apart = N > 4 * near || ((N - near) * 256 > near * tk && (N - near) * (Hq / Hk) > 32 * SINK_ITEMS);
    pl.sink_keys = w >= 0 && S > 0 && apart ? ((S < N ? S : N) + 31) / 32 * 32 : 0;
    if ((long)B * Hk * pl.sink_keys >= (1L << 22)) pl.sink_keys = 0;     // (their sum would be more than 2^32 threads)
    pl.chunks = pl.per_chunk = pl.shares = 0;
    if (pl.sink_keys) {
        // workgroups of waves that share the 32 keys and have their own queries each, about 1024 waves in all and 2 tiles or more a
        // workgroup: all of q and do is read once (16384 tokens x 16 heads of 128, 134 MB: 36 us; one-wave workgroups 34; 3 x
        // 1001 x 8 heads in groups of 4, fp32: the backward 264 us against 293)
        const int waves = sink_waves(pl.dp * (dtype == VITK_F32 ? 4 : 2)), rows = 32 * waves;
        const long items = (long)((N + rows - 1) / rows) * (Hq / Hk), sets = (long)B * Hk * (pl.sink_keys / 32);
        const long want = (1024 / waves + sets - 1) / sets, per = std::max((items + want - 1) / want, 2L);
        pl.per_chunk = (int)per;
        pl.chunks = (int)((items + per - 1) / per);
        pl.shares = pl.chunks * waves;
    }
    return pl;
}
// a number for each of N rows or groups in the workspace
long stat_floats(int B, int Hq, int N) { return ((long)B * Hq * N + 3) / 4 * 4; }
long part_floats(const Plan& pl, int B, int Hk) { return (long)B * Hk * (pl.sink_keys / 32) * pl.shares * 2 * pl.dp * 32; }

int check_window(const char* what, int dtype, int B, int N, int Hq, int Hk, int dh, float scale, int sinks) {
    VITK_CHECK_ARG(dtype == VITK_F32 || dtype == VITK_BF16, "%s: bad dtype %d", what, dtype);
    VITK_CHECK_ARG(B >= 0 && N >= 0 && N < (1 << 28) && Hq >= 1 && Hk >= 1, "%s: bad shape B=%d N=%d Hq=%d Hk=%d", what, B, N, Hq, Hk);
    VITK_CHECK_ARG(Hq % Hk == 0, "%s: %d query heads are no multiple of %d key heads", what, Hq, Hk);
    VITK_CHECK_ARG(dh >= 8 && dh <= 128 && dh % 8 == 0, "%s: head width %d must be a multiple of 8 up to 128", what, dh);
    VITK_CHECK_ARG(scale > 0.f && scale < INFINITY, "%s: the scale must be positive and finite", what);
    VITK_CHECK_ARG(sinks >= 0, "%s: bad number of sinks %d", what, sinks);
    // two threads a row, at most 2^32 a launch
    VITK_CHECK_ARG((long)B * Hq * (N + 256L) < (1L << 31), "%s: B * Hq * N = %ld rows are too many for one call", what, (long)B * Hq * N);
    return VITK_OK;
}
int check_view(const char* what, const char* name, const View& v, int dtype) {
    const int per = dtype == VITK_F32 ? 4 : 8;
    VITK_CHECK_ARG(v.p && (reinterpret_cast<uintptr_t>(v.p) & 15) == 0 && v.sb % per == 0 && v.sn % per == 0 && v.sh % per == 0,
                   "%s: %s must be 16-byte aligned, its strides too", what, name);
    VITK_CHECK_ARG(v.sn >= 0 && v.sn < (1L << 20) * per, "%s: the tokens of %s are too far apart", what, name);    // 128 rows under 2 GiB
    return VITK_OK;
}
void fill_params(WindowParams& p, int B, int N, int Hq, int Hk, int dh, int w, int S, int causal, float scale, const int* lengths) {
    p.lengths = lengths;
    p.B = B; p.N = N; p.Hq = Hq; p.Hk = Hk; p.G = Hq / Hk; p.dh = dh;
    p.w = w < 0 || w >= N - 1 ? -1 : w;                  // a window that covers the sequence is no window
    p.S = p.w < 0 ? 0 : (S < N ? S : N);
    p.causal = causal != 0;
    p.scale = scale;
    p.sc2 = scale * 1.4426950408889634f;
}
// Sets the order of the (tile, sequence, key head) pieces of `each` neighbours, and the grid that goes with it.  By tile, the long
// ones first, dealt to the XCDs in turn: where pieces differ (sequences of different lengths, causal rows without a window:
// 8192 tokens x 16 heads of 128, groups of 4, forward and backward 298 + 1265 us; an eighth of them in a row to each XCD, some of
// which then had all the long ones, 395 + 1795), and where heads are a multiple of 8, so that a head stays on one XCD (16 x 577 x
// 12 heads of 64, window 64: 21 + 65 us against 23 + 74).  A multiple of 8 heads whose tiles differ by the sequence alone: whole
// heads to each XCD in turn (1001, 100 and 1001 tokens x 16 heads of 80, fp32: 137 + 418 us against 186 + 570 by tile).  Else an
// eighth of the pieces in a row to each XCD (16384 tokens, groups of 4 heads of 128, window 1024: 180 + 576 us against 185 + 586).
unsigned xcd_grid(WindowParams& p, int tiles, int each, bool by_tile) {
    const int heads = p.B * p.Hk, total = heads * tiles * each;
    p.total = total;
    p.by_tile = by_tile;
    p.inner = by_tile ? heads : tiles;
    p.run = by_tile ? each : (p.lengths && heads % 8 == 0 ? tiles * each : (total + 7) / 8);
    const long round = 8L * p.run;
    return (unsigned)((total + round - 1) / round * round);
}
bool by_tile(const WindowParams& p) {
    const bool eights = (long)p.B * p.Hk % 8 == 0;
    if (p.w < 0 && !p.causal && p.lengths && eights) return false;
    return p.lengths || (p.causal && p.w < 0) || eights;
}

constexpr int NW = 4;
// bytes of LDS that `waves` groups of 32 rows need to leave through (put_rows), after which `n` accumulators of theirs were joined
template <typename T, int DP> size_t rows_lds(int groups, int n) {
    const size_t rows = 32 * groups * WCfg<T, DP>::LD * sizeof(T), join = n ? (size_t)groups * (DP / 2 * n + 2) * 64 * sizeof(float) : 0;
    return rows > join ? rows : join;
}
template <typename T, int HW, int KS, int BK, bool FINE = false> void run_fwd_tiles(WindowParams p, hipStream_t st) {
    constexpr int DP = (HW + 31) / 32 * 32, WPE = sizeof(T) == 4 && DP == 128 ? 1 : 2, RG = NW / KS;             // one wave a SIMD where two would spill
    p.tiles = (p.N + 32 * RG - 1) / (32 * RG);
    const unsigned grid = xcd_grid(p, p.tiles, p.G, by_tile(p));
    const size_t lds = std::max<size_t>(4 * BK * DP * sizeof(T), rows_lds<T, DP>(RG, KS - 1));
    vitk_lds_optin(reinterpret_cast<const void*>(&window_fwd_kernel<T, HW, NW, KS, BK, WPE, FINE>), lds);
    hipLaunchKernelGGL((window_fwd_kernel<T, HW, NW, KS, BK, WPE, FINE>), dim3(grid), dim3(64 * NW), lds, st, p);
}
// Key tiles of 64 in bf16; of 32 where the window is narrow and a tile of 64 would be mostly edge (16 x 577 tokens x 12 heads of
// 64, window 64 on both sides: 22.9 us against 25.6, window 256: 30.7 against 31.4; 2 x 8192 x 16 heads of 128, causal window
// of 512: 131 against 126, 16384 x 16, of 1024: 200 against 186).
template <typename T, int HW> void run_fwd(const WindowParams& p, const Plan& pl, hipStream_t st) {
    if constexpr (sizeof(T) == 2) {
        if (pl.fine) return run_fwd_tiles<T, HW, 2, 64, true>(p, st);
    }
    if (pl.halves_q) return run_fwd_tiles<T, HW, 2, 64>(p, st);
    if constexpr (sizeof(T) == 2) {
        if (p.w < 0 || p.w > NARROW) return run_fwd_tiles<T, HW, 1, 64>(p, st);
    }
    run_fwd_tiles<T, HW, 1, 32>(p, st);
}
template <typename T, int HW, int KS, bool FINE> void run_dq(WindowParams p, hipStream_t st) {
    constexpr int DP = (HW + 31) / 32 * 32, BK = 32 * KS, WPE = sizeof(T) == 4 && DP == 128 ? 1 : 2, RG = NW / KS;
    p.tiles = (p.N + 32 * RG - 1) / (32 * RG);
    const unsigned grid = xcd_grid(p, p.tiles, p.G, by_tile(p));
    const size_t lds = std::max<size_t>(4 * BK * DP * sizeof(T), rows_lds<T, DP>(RG, KS - 1));
    vitk_lds_optin(reinterpret_cast<const void*>(&window_dq_kernel<T, HW, NW, KS, BK, WPE, FINE>), lds);
    hipLaunchKernelGGL((window_dq_kernel<T, HW, NW, KS, BK, WPE, FINE>), dim3(grid), dim3(64 * NW), lds, st, p);
}
template <typename T, int HW, int W, int KS, int BQ, bool SINK, bool FINE> void run_dkv(WindowParams p, int keys, hipStream_t st) {
    constexpr int DP = (HW + 31) / 32 * 32;
    // V rows in LDS where they, K's and both accumulators do not fit the registers of two waves a SIMD
    constexpr bool VLDS = sizeof(T) == 2 && DP >= 96 && !SINK;
    constexpr int WPE = (sizeof(T) == 4 && DP >= 96) || SINK || (FINE && DP == 128) ? 1 : 2, RG = W / KS;
    p.tiles = (keys + 32 * RG - 1) / (32 * RG);
    p.heavy = SINK ? 0 : (p.S > p.key0 ? (p.S - p.key0 + 32 * RG - 1) / (32 * RG) : 0);
    if (p.heavy >= p.tiles) p.heavy = 0;                 // nothing but sinks: all alike
    const unsigned grid = xcd_grid(p, p.tiles - p.heavy, SINK ? p.chunks : 1, !SINK && by_tile(p)) + (p.heavy * p.B * p.Hk + 7) / 8 * 8;
    const size_t tl = 4 * BQ * DP * sizeof(T) + 4 * BQ * sizeof(float) + (VLDS ? 32 * RG * DP * sizeof(T) : 0);
    const size_t lds = std::max<size_t>(tl, rows_lds<T, DP>(RG, 2 * (KS - 1)));
    vitk_lds_optin(reinterpret_cast<const void*>(&window_dkv_kernel<T, HW, W, KS, BQ, SINK, VLDS, WPE, FINE>), lds);
    hipLaunchKernelGGL((window_dkv_kernel<T, HW, W, KS, BQ, SINK, VLDS, WPE, FINE>), dim3(grid), dim3(64 * W), lds, st, p);
}
template <typename T, int HW, bool FINE> void run_bwd(WindowParams p, const Plan& pl, void* dq, hipStream_t st) {
    constexpr int DP = (HW + 31) / 32 * 32, BQ = sizeof(T) == 2 && DP <= 64 ? 64 : 32;
    p.out = dq;
    if constexpr (!FINE) {
        if (!pl.halves_q) run_dq<T, HW, 1, FINE>(p, st);
    }
    if (pl.halves_q) run_dq<T, HW, 2, FINE>(p, st);
    if (pl.sink_keys) {
        WindowParams s = p;
        s.key0 = 0;
        s.chunks = pl.chunks;
        s.per_chunk = pl.per_chunk;
        constexpr int W = sink_waves(DP * sizeof(T));
        run_dkv<T, HW, W, W, 32 * W, true, FINE>(s, pl.sink_keys, st);
        s.tiles = pl.sink_keys / 32;
        s.chunks = pl.shares;
        hipLaunchKernelGGL((window_sink_sum_kernel<T, DP>), dim3((unsigned)((long)p.B * p.Hk * s.tiles * 2 * (DP / 2))), dim3(256),
                           0, st, s);
    }
    p.key0 = pl.sink_keys;
    const int rest = p.N - pl.sink_keys;
    if (rest <= 0) return;
    if constexpr (!FINE) {
        if (!pl.halves_k) run_dkv<T, HW, NW, 1, BQ, false, FINE>(p, rest, st);
    }
    if (pl.halves_k) run_dkv<T, HW, NW, 2, 64, false, FINE>(p, rest, st);
}
template <typename T, int HW> void run_bwd(const WindowParams& p, const Plan& pl, void* dq, hipStream_t st) {
    if constexpr (sizeof(T) == 2) {
        if (pl.fine) return run_bwd<T, HW, true>(p, pl, dq, st);
    }
    run_bwd<T, HW, false>(p, pl, dq, st);
}

}  // namespace

extern "C" int vitk_window_attn_fwd(int dtype, int B, int N, int Hq, int Hk, int dh, const void* q, long qb, long qn, long qh,
                                    const void* k, long kb, long kn, long kh, const void* v, long vb, long vn, long vh, float scale,
                                    int window, int sinks, int causal, const int* lengths, void* out, void* out_lo, float* lse,
                                    hipStream_t stream) {
    const char* what = "vitk_window_attn_fwd";
    if (int e = check_window(what, dtype, B, N, Hq, Hk, dh, scale, sinks)) return e;
    if (B == 0 || N == 0) return VITK_OK;
    WindowParams p = {};
    if (N == 1) qn = kn = vn = 0;                        // one token: whatever its stride is, nobody goes there
    p.q = View{q, qb, qn, qh};
    p.k = View{k, kb, kn, kh};
    p.v = View{v, vb, vn, vh};
    if (int e = check_view(what, "q", p.q, dtype)) return e;
    if (int e = check_view(what, "k", p.k, dtype)) return e;
    if (int e = check_view(what, "v", p.v, dtype)) return e;
    VITK_CHECK_ARG(out && ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(out_lo)) & 15) == 0,
                   "%s: out must be 16-byte aligned", what);
    fill_params(p, B, N, Hq, Hk, dh, window, sinks, causal, scale, lengths);
    p.out = out;
    p.o_lo = out_lo;
    p.lse = lse;
    const Plan pl = make_plan(dtype, B, N, Hq, Hk, dh, p.w, p.S, p.causal, p.causal || p.w >= 0 || lengths);
#define GO(T, D) run_fwd<T, D>(p, pl, stream)
#define BY_WIDTH(T) switch (pl.width) { case 32: GO(T, 32); break; case 64: GO(T, 64); break; case 80: GO(T, 80); break; \
                                       case 96: GO(T, 96); break; default: GO(T, 128); break; }
    if (dtype == VITK_BF16) { BY_WIDTH(__bf16) }
    else { BY_WIDTH(float) }
#undef GO
    VITK_CHECK_LAUNCH(what);
    return VITK_OK;
}

extern "C" long vitk_window_attn_bwd_workspace_bytes(int dtype, int B, int N, int Hq, int Hk, int dh, int window, int sinks) {
    if (B <= 0 || N <= 0 || Hq <= 0 || Hk <= 0 || Hq % Hk || dh < 8 || dh > 128 || sinks < 0) return 0;
    WindowParams p = {};
    fill_params(p, B, N, Hq, Hk, dh, window, sinks, 0, 1.f, nullptr);
    long part = 0;                                       // causal or not, whichever leaves more
    for (int causal = 0; causal < 2; ++causal)
        part = std::max(part, part_floats(make_plan(dtype, B, N, Hq, Hk, dh, p.w, p.S, causal, true), B, Hk));
    return (2 * stat_floats(B, Hq, N) + stat_floats(B, Hq, (N + 31) / 32)) * 4 + part * 4;
}

extern "C" int vitk_window_attn_bwd(int dtype, int B, int N, int Hq, int Hk, int dh, const void* q, long qb, long qn, long qh,
                                    const void* k, long kb, long kn, long kh, const void* v, long vb, long vn, long vh, float scale,
                                    int window, int sinks, int causal, const int* lengths, const void* out, const void* out_lo, const float* lse,
                                    const void* dout, long ob, long on, long oh, void* dq, void* dk, void* dv, void* workspace,
                                    hipStream_t stream) {
    const char* what = "vitk_window_attn_bwd";
    if (int e = check_window(what, dtype, B, N, Hq, Hk, dh, scale, sinks)) return e;
    if (B == 0 || N == 0) return VITK_OK;
    WindowParams p = {};
    if (N == 1) qn = kn = vn = 0;                        // one token: whatever its stride is, nobody goes there
    p.q = View{q, qb, qn, qh};
    p.k = View{k, kb, kn, kh};
    p.v = View{v, vb, vn, vh};
    p.dout = View{dout, ob, N == 1 ? 0 : on, oh};
    if (int e = check_view(what, "q", p.q, dtype)) return e;
    if (int e = check_view(what, "k", p.k, dtype)) return e;
    if (int e = check_view(what, "v", p.v, dtype)) return e;
    if (int e = check_view(what, "dout", p.dout, dtype)) return e;
    VITK_CHECK_ARG(out && lse && dq && dk && dv && workspace, "%s: null pointer", what);
    VITK_CHECK_ARG(((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(out_lo) | reinterpret_cast<uintptr_t>(dq) | reinterpret_cast<uintptr_t>(dk) |
                     reinterpret_cast<uintptr_t>(dv) | reinterpret_cast<uintptr_t>(workspace)) & 15) == 0,
                   "%s: out, dq, dk, dv and the workspace must be 16-byte aligned", what);
    fill_params(p, B, N, Hq, Hk, dh, window, sinks, causal, scale, lengths);
    p.o = out;
    p.o_lo = const_cast<void*>(out_lo);
    p.lse = const_cast<float*>(lse);
    p.delta = static_cast<float*>(workspace);
    p.shift = p.delta + stat_floats(B, Hq, N);
    p.far = reinterpret_cast<int*>(p.shift + stat_floats(B, Hq, N));
    p.part = p.shift + stat_floats(B, Hq, N) + stat_floats(B, Hq, (N + 31) / 32);
    p.dk = dk;
    p.dv = dv;
    const Plan pl = make_plan(dtype, B, N, Hq, Hk, dh, p.w, p.S, p.causal, p.causal || p.w >= 0 || lengths);
#define GO(T, D) run_bwd<T, D>(p, pl, dq, stream)
    if (dtype == VITK_BF16) { BY_WIDTH(__bf16) }
    else { BY_WIDTH(float) }
#undef GO
#undef BY_WIDTH
    VITK_CHECK_LAUNCH(what);
    return VITK_OK;
}
