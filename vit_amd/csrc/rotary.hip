// Rotary positions and the per-head RMS norm of queries and keys with the rotation in the same pass.
//
//   table[p][i] = m (cos, sin)(pos[p][axis(i)] * freq[i])        angles and their sines in 64 bits, stored in 32
//   rotary      : y1 = x1 c - x2 s,  y2 = x2 c + x1 s  over pairs (i, i + rot/2) or (2i, 2i + 1); d >= rot unchanged;
//                 the adjoint is the same map with s -> -s
//   qk_norm     : y = R (g x r),  r = 1 / sqrt(mean x^2 + eps)
//   backward    : u = R^T dy,  t = u g,  dx = r (t - x r^2 mean(t x)),  dg = sum over rows of u x r
//
// All of it is bound by memory: every element is read and written once (the backward reads x and dy), and the table,
// a few hundred bytes a token, is shared by the token's heads.  Layout of the work: a "unit" is V pairs, i.e. two
// chunks of V elements of one row, so both members of each pair sit in one lane whatever the layout of the pairs.  V is
// 16 bytes' worth where the row's shape and alignment allow it, else 8 bytes' worth, else one element.
#include <type_traits>
#include "common.h"

namespace vitk {

template <typename T, int V> struct Chunk;                // V elements as one load / store
template <> struct Chunk<__bf16, 8> { typedef u32x4 R; };
template <> struct Chunk<__bf16, 4> { typedef u32x2 R; };
template <> struct Chunk<__bf16, 1> { typedef unsigned short R; };
template <> struct Chunk<float, 4> { typedef u32x4 R; };
template <> struct Chunk<float, 2> { typedef u32x2 R; };
template <> struct Chunk<float, 1> { typedef float R; };

template <typename T, int V> __device__ __forceinline__ typename Chunk<T, V>::R chunk_load(const T* p) {
    return *reinterpret_cast<const typename Chunk<T, V>::R*>(p);
}
template <typename T, int V> __device__ __forceinline__ void chunk_unpack(const typename Chunk<T, V>::R& r, float* f) {
    struct A { T e[V]; };
    const A a = __builtin_bit_cast(A, r);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = (float)a.e[i];
}
template <typename T, int V> __device__ __forceinline__ void chunk_store(T* p, const float* f) {
    struct A { T e[V]; };
    A a;
#pragma unroll
    for (int i = 0; i < V; ++i) a.e[i] = (T)f[i];         // the one rounding of the result
    *reinterpret_cast<typename Chunk<T, V>::R*>(p) = __builtin_bit_cast(typename Chunk<T, V>::R, a);
}

struct Pos {                  // which table row a token takes
    const void* ids;          // [B*N] int32 / int64, or NULL: row offset + n
    int ids64;
    long offset;
    long rows;                // rows of the table; an id outside of it gives NaN in the rotated part
};
__device__ __forceinline__ long pos_row(const Pos& p, long bn, int n) {
    if (!p.ids) return p.offset + n;
    return p.ids64 ? (long)static_cast<const long long*>(p.ids)[bn] : (long)static_cast<const int*>(p.ids)[bn];
}

// n (cos, sin) pairs from pair `at` of a table row on
template <int N> __device__ __forceinline__ void load_pairs(const float* row, int at, float* c, float* s) {
    const float* t = row + 2 * at;
    if (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const f32x4 w = *reinterpret_cast<const f32x4*>(t + 2 * i);
            c[i] = w[0]; s[i] = w[1]; c[i + 1] = w[2]; s[i + 1] = w[3];
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) { c[i] = t[2 * i]; s[i] = t[2 * i + 1]; }
    }
}

// A unit's two chunks are V elements at u and V elements half the rotated width further on, whichever way the pairs lie: a
// chunk with its partner (halves), or two chunks of V / 2 pairs each (interleaved), so that neighbouring lanes read
// neighbouring chunks either way.  (Single elements, interleaved: the pair itself.)
template <int V, bool INTER> __device__ __forceinline__ void load_turn(const float* table, long row, long rows, int pairs, int u, float* c, float* s) {
    if (row < 0 || row >= rows) {
#pragma unroll
        for (int i = 0; i < V; ++i) c[i] = s[i] = __builtin_nanf("");
        return;
    }
    const float* t = table + 2 * row * pairs;
    if (INTER && V > 1) {
        load_pairs<V / 2>(t, V / 2 * u, c, s);
        load_pairs<V / 2>(t, pairs / 2 + V / 2 * u, c + V / 2, s + V / 2);
    } else {
        load_pairs<V>(t, V * u, c, s);
    }
}

// f[0..V) and f[V..2V): the unit's two chunks
template <int V, bool INTER> __device__ __forceinline__ void turn(float* f, const float* c, const float* s) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int a = INTER ? 2 * i : i, b = INTER ? 2 * i + 1 : V + i;
        const float x = f[a], y = f[b];
        f[a] = x * c[i] - y * s[i];
        f[b] = y * c[i] + x * s[i];
    }
}

// element offsets of a unit's two chunks within the row; n2: whether the second one exists (an unrotated tail may have an odd
// number of chunks)
template <int V, bool INTER> __device__ __forceinline__ void unit_at(int u, int urot, int units, int rot, int dh, int& d0, int& d1, bool& n2) {
    n2 = true;
    if (u < urot) {
        d0 = INTER && V == 1 ? 2 * u : V * u;
        d1 = INTER && V == 1 ? d0 + 1 : d0 + rot / 2;
    } else {
        d0 = rot + V * (u - urot);
        d1 = d0 + V * (units - urot);
        n2 = d1 < dh;
    }
}

// ------------------------------------------------------------------------------------------------------- the table
struct Freqs { double f[128]; };
template <typename P>
__global__ __launch_bounds__(256) void rotary_table_kernel(const Freqs fr, const P* __restrict__ pos, int axes, long rows, int pairs,
                                                           int per_axis, double mul, float* __restrict__ out) {
    const long total = rows * pairs;
    for (long e = (long)blockIdx.x * 256 + threadIdx.x; e < total; e += (long)gridDim.x * 256) {
        const long p = e / pairs;
        const int i = (int)(e - p * pairs);
        const int a = i / per_axis;
        double sn, cs;
        sincos((double)pos[p * axes + a] * fr.f[i - a * per_axis], &sn, &cs);
        out[2 * e] = (float)(mul * cs);
        out[2 * e + 1] = (float)(mul * sn);
    }
}

// ------------------------------------------------------------------------------------------------------ the rotation
struct RotaryParams {
    const void* x;
    void* y;
    long sb, sn, sh;                       // x: element (b, n, h, d) at b*sb + n*sn + h*sh + d; y: [B][N][H][dh]
    const float* table;
    Pos pos;
    int N, H, dh, rot, urot, units, hgroups;
    unsigned total;                        // B * N * hgroups * units
    float sgn;                             // +1, or -1: the adjoint
};

// A lane keeps its unit's turn in registers and applies it to HPT heads of the token, all of whose loads are in flight
// at once.  32 x 577 x 12 heads of 64, bf16: 11.7 us for 57 MB (out of the last-level cache); 16411 x 16 heads of 80, fp32, half of
// it turned: 44 us for 169 MB, 3.8 TB/s, where a copy of 4 GiB does 4.8.
template <typename T, int V, bool INTER, int HPT>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryParams p) {
    const unsigned id = blockIdx.x * 256u + threadIdx.x;
    if (id >= p.total) return;
    const unsigned r = id / (unsigned)p.units;
    const int u = (int)(id - r * p.units);
    const unsigned bn = r / (unsigned)p.hgroups;
    const int h0 = (int)(r - bn * p.hgroups) * HPT;
    const unsigned b = bn / (unsigned)p.N;
    const int n = (int)(bn - b * p.N);
    const T* x = static_cast<const T*>(p.x) + (long)b * p.sb + (long)n * p.sn + (long)h0 * p.sh;
    T* y = static_cast<T*>(p.y) + ((long)bn * p.H + h0) * p.dh;
    int d0, d1;
    bool n2;
    unit_at<V, INTER>(u, p.urot, p.units, p.rot, p.dh, d0, d1, n2);
    typename Chunk<T, V>::R a[HPT], c2[HPT];
#pragma unroll
    for (int k = 0; k < HPT; ++k)
        if (h0 + k < p.H) {
            a[k] = chunk_load<T, V>(x + k * p.sh + d0);
            if (n2) c2[k] = chunk_load<T, V>(x + k * p.sh + d1);
        }
    float c[V], s[V];
    if (u < p.urot) {
        load_turn<V, INTER>(p.table, pos_row(p.pos, bn, n), p.pos.rows, p.rot / 2, u, c, s);
#pragma unroll
        for (int i = 0; i < V; ++i) s[i] *= p.sgn;
    }
#pragma unroll
    for (int k = 0; k < HPT; ++k)
        if (h0 + k < p.H) {
            T* o = y + (long)k * p.dh;
            if (u < p.urot) {
                float f[2 * V];
                chunk_unpack<T, V>(a[k], f);
                chunk_unpack<T, V>(c2[k], f + V);
                turn<V, INTER>(f, c, s);
                chunk_store<T, V>(o + d0, f);
                chunk_store<T, V>(o + d1, f + V);
            } else {
                *reinterpret_cast<typename Chunk<T, V>::R*>(o + d0) = a[k];
                if (n2) *reinterpret_cast<typename Chunk<T, V>::R*>(o + d1) = c2[k];
            }
        }
}

// --------------------------------------------------------------------------------------------- norm and rotation
struct Side {                              // queries or keys
    const void* x;
    long sb, sn, sh;
    const void* dy;                        // backward: the gradient, with its own strides
    long gb, gn, gh;
    const float* gamma;                    // [dh] or NULL
    void* y;                               // forward: [B][N][H][dh]; backward: dx, the same
    float* part;                           // backward: gamma's partial sums [blocks][dh], or NULL
    int H, hgroups;                        // hgroups = ceil(H / HPT)
    unsigned blocks;                       // workgroups of this side
    unsigned groups;                       // B * N * hgroups
};
struct QkNormParams {
    Side q, k;
    const float* table;
    Pos pos;
    int N, dh, rot, urot, units, lpr_log2; // a row takes 2^lpr_log2 lanes, `units` of them at work
    float eps;
};

// sum over the row's lanes, in every one of them: lane exchanges on the vector unit (a shuffle would go through LDS)
__device__ __forceinline__ float row_sum(float v, int lpr_log2) {
    auto dpp = [](float x, auto ctrl) {
        return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, 0xf, 0xf, true));
    };
    if (lpr_log2 > 0) v += dpp(v, std::integral_constant<int, 0xB1>{});      // quad_perm [1,0,3,2]
    if (lpr_log2 > 1) v += dpp(v, std::integral_constant<int, 0x4E>{});      // quad_perm [2,3,0,1]
    if (lpr_log2 > 2) v += dpp(v, std::integral_constant<int, 0x141>{});     // row_half_mirror: the other four of eight
    if (lpr_log2 > 3) v += dpp(v, std::integral_constant<int, 0x140>{});     // row_mirror: the other eight of sixteen
    if (lpr_log2 > 4) v += __shfl_xor(v, 16, 64);
    if (lpr_log2 > 5) v += __shfl_xor(v, 32, 64);
    return v;
}

// One row (token, head) on 2^lpr_log2 lanes, 256 >> lpr_log2 of them side by side in a workgroup; a lane group takes HPT
// heads of one token in a step, so that the token's turn, 8 bytes a pair against 4 or 8 of x, is read once for HPT rows.
// BWD walks several steps per workgroup so that gamma's sum stays in registers and ends in one partial row per workgroup (a
// second kernel adds those in a fixed order: no atomics).  128 x 197 x (12 + 12) heads of 64, bf16: forward 31 us, backward 58 +
// 6, for 155 and 232 MB (5.0 and 4.0 TB/s); 32769 x (16 + 4) heads of 80, fp32: 87 us, 130 + 7, for 419 and 629 MB (4.8 TB/s, a large
// copy's rate).
template <typename T, int V, bool INTER, int HPT, bool BWD>
__global__ __launch_bounds__(256) void qk_norm_kernel(const QkNormParams p) {
    const bool isq = blockIdx.x < p.q.blocks;
    const Side& S = isq ? p.q : p.k;
    const unsigned blk = isq ? blockIdx.x : blockIdx.x - p.q.blocks;
    const int rows = 256 >> p.lpr_log2;
    const int u = threadIdx.x & ((1 << p.lpr_log2) - 1), slot = threadIdx.x >> p.lpr_log2;
    const bool live = u < p.units;
    int d0 = 0, d1 = 0;
    bool n2 = false;
    if (live) unit_at<V, INTER>(u, p.urot, p.units, p.rot, p.dh, d0, d1, n2);
    float g[2 * V], acc[2 * V];
#pragma unroll
    for (int i = 0; i < 2 * V; ++i) {
        g[i] = !live || (i >= V && !n2) ? 0.f : (S.gamma ? S.gamma[(i < V ? d0 : d1 - V) + i] : 1.f);
        acc[i] = 0.f;
    }
    const float inv = 1.f / (float)p.dh;
    // the loop's bounds are the same for every lane of the workgroup: the shuffles below need them all
    for (unsigned base = blk * rows; base < S.groups; base += S.blocks * rows) {
        const unsigned grp = base + slot;
        const bool on = live && grp < S.groups;
        const unsigned bn = grp / (unsigned)S.hgroups;
        const int h0 = (int)(grp - bn * S.hgroups) * HPT;
        const unsigned b = bn / (unsigned)p.N;
        const int n = (int)(bn - b * p.N);
        typename Chunk<T, V>::R a[HPT] = {}, c2[HPT] = {}, ga[HPT] = {}, gc[HPT] = {};
        float c[V], s[V];
        if (on) {
            const T* x = static_cast<const T*>(S.x) + (long)b * S.sb + (long)n * S.sn + (long)h0 * S.sh;
            const T* dy = BWD ? static_cast<const T*>(S.dy) + (long)b * S.gb + (long)n * S.gn + (long)h0 * S.gh : nullptr;
#pragma unroll
            for (int k = 0; k < HPT; ++k)
                if (h0 + k < S.H) {
                    a[k] = chunk_load<T, V>(x + k * S.sh + d0);
                    if (n2) c2[k] = chunk_load<T, V>(x + k * S.sh + d1);
                    if (BWD) {
                        ga[k] = chunk_load<T, V>(dy + k * S.gh + d0);
                        if (n2) gc[k] = chunk_load<T, V>(dy + k * S.gh + d1);
                    }
                }
            if (u < p.urot) load_turn<V, INTER>(p.table, pos_row(p.pos, bn, n), p.pos.rows, p.rot / 2, u, c, s);
            if (BWD) {
#pragma unroll
                for (int i = 0; i < V; ++i) s[i] = -s[i];
            }
        }
#pragma unroll
        for (int k = 0; k < HPT; ++k) {
            float f[2 * V], ss = 0.f;
            chunk_unpack<T, V>(a[k], f);
            chunk_unpack<T, V>(c2[k], f + V);
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) ss += f[i] * f[i];
            ss = row_sum(ss, p.lpr_log2);
            const float r = 1.f / sqrtf(ss * inv + p.eps);
            T* o = static_cast<T*>(S.y) + ((long)bn * S.H + h0 + k) * p.dh;
            const bool st = on && h0 + k < S.H;
            if (!BWD) {
#pragma unroll
                for (int i = 0; i < 2 * V; ++i) f[i] = f[i] * r * g[i];
                if (st) {
                    if (u < p.urot) turn<V, INTER>(f, c, s);
                    chunk_store<T, V>(o + d0, f);
                    if (n2) chunk_store<T, V>(o + d1, f + V);
                }
            } else {
                float w[2 * V], tx = 0.f;
                chunk_unpack<T, V>(ga[k], w);
                chunk_unpack<T, V>(gc[k], w + V);
                if (on && u < p.urot) turn<V, INTER>(w, c, s);
#pragma unroll
                for (int i = 0; i < 2 * V; ++i) {
                    if (st) acc[i] += w[i] * f[i] * r;
                    w[i] *= g[i];
                    tx += w[i] * f[i];
                }
                tx = row_sum(tx, p.lpr_log2);
                const float cf = tx * inv * r * r;
#pragma unroll
                for (int i = 0; i < 2 * V; ++i) w[i] = r * (w[i] - f[i] * cf);
                if (st) {
                    chunk_store<T, V>(o + d0, w);
                    if (n2) chunk_store<T, V>(o + d1, w + V);
                }
            }
        }
    }
    if (BWD && S.part) {
        // gamma's sums of the workgroup's lanes: over the slots of one unit, in order, by the threads (part, unit, element)
        __shared__ float red[2 * V][256];
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) red[i][threadIdx.x] = acc[i];
        __syncthreads();
        for (int e = threadIdx.x; e < 2 * V << p.lpr_log2; e += 256) {
            const int i = e >> p.lpr_log2, uu = e & ((1 << p.lpr_log2) - 1);
            if (uu >= p.units) continue;
            int a0, a1;
            bool two;
            unit_at<V, INTER>(uu, p.urot, p.units, p.rot, p.dh, a0, a1, two);
            if (i >= V && !two) continue;
            float t = 0.f;
            for (int w = 0; w < rows; ++w) t += red[i][(w << p.lpr_log2) + uu];
            S.part[(long)blk * p.dh + (i < V ? a0 : a1 - V) + i] = t;
        }
    }
}

// dgamma[side][d] = sum over the workgroups' partial rows, in an order that the sizes alone fix
__global__ __launch_bounds__(256) void qk_norm_dgamma_kernel(const float* pq, const float* pk, unsigned nq, unsigned nk, int dh,
                                                             float* dgq, float* dgk) {
    const float* part = blockIdx.y ? pk : pq;
    float* out = blockIdx.y ? dgk : dgq;
    const unsigned nb = blockIdx.y ? nk : nq;
    if (!out) return;
    const int col = blockIdx.x * 16 + (threadIdx.x & 15), row = threadIdx.x >> 4;
    __shared__ float red[16][17];
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (col < dh) {
        unsigned r = row;
        for (; r + 48 < nb; r += 64)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] += part[(long)(r + 16 * e) * dh + col];
        for (; r < nb; r += 16) s[0] += part[(long)r * dh + col];
    }
    red[row][threadIdx.x & 15] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    if (row == 0 && col < dh) {
        float t = 0.f;
        for (int r = 0; r < 16; ++r) t += red[r][threadIdx.x & 15];
        out[col] = t;
    }
}

}  // namespace vitk

using namespace vitk;

namespace {

bool aligned(const void* p, long sb, long sn, long sh, int esize, int bytes) {
    return (reinterpret_cast<uintptr_t>(p) % bytes) == 0 && (sb * esize) % bytes == 0 && (sn * esize) % bytes == 0 &&
           (sh * esize) % bytes == 0;
}
// elements per chunk: as wide as the row's shape and every operand's alignment allow (1 always does)
int chunk_elems(int esize, int dh, int rot, bool al16, bool al8) {
    const int v16 = 16 / esize, v8 = 8 / esize;
    if (al16 && (rot / 2) % v16 == 0 && dh % v16 == 0) return v16;
    if (al8 && (rot / 2) % v8 == 0 && dh % v8 == 0) return v8;
    return 1;
}
int check_pos(const char* what, const float* table, long rows, int N, int rot, int dh, const void* ids, long offset) {
    VITK_CHECK_ARG(rot >= 0 && rot % 2 == 0 && rot <= dh, "%s: rotated width %d must be even and at most the head width %d", what, rot, dh);
    if (rot == 0) return VITK_OK;
    VITK_CHECK_ARG(table && (reinterpret_cast<uintptr_t>(table) & 15) == 0, "%s: the table must be 16-byte aligned", what);
    VITK_CHECK_ARG(ids || (offset >= 0 && offset <= rows - N), "%s: %d tokens from row %ld on are outside the table's %ld rows", what, N,
                   offset, rows);
    return VITK_OK;
}

template <typename T, int V>
void launch_rotary(const RotaryParams& p, bool inter, bool wide, hipStream_t st) {
    const unsigned blocks = (p.total + 255) / 256;
#define GO(I, H) hipLaunchKernelGGL((rotary_kernel<T, V, I, H>), dim3(blocks), dim3(256), 0, st, p)
    if (inter) { if (wide) GO(true, 4); else GO(true, 1); }
    else { if (wide) GO(false, 4); else GO(false, 1); }
#undef GO
}
// heads a lane takes in a step: as below where the call is large, one where it is small and a step's latency counts
constexpr int HEADS_FWD = 4, HEADS_BWD = 2;
template <typename T, int V, bool BWD>
void launch_qk_norm(const QkNormParams& p, bool inter, int hpt, hipStream_t st) {
    const unsigned blocks = p.q.blocks + p.k.blocks;
    constexpr int W = BWD ? HEADS_BWD : HEADS_FWD;
#define GO(I, H) hipLaunchKernelGGL((qk_norm_kernel<T, V, I, H, BWD>), dim3(blocks), dim3(256), 0, st, p)
    if (inter) { if (hpt > 1) GO(true, W); else GO(true, 1); }
    else { if (hpt > 1) GO(false, W); else GO(false, 1); }
#undef GO
}

constexpr unsigned NORM_BLOCKS = 1024;     // backward: workgroups of each side at most, one partial row each

bool large_norm(long B, long N, long H, long dh) { return B * N * H * dh >= 256L * 256 * 64; }     // 64 elements for each of 256 lanes a CU

// the parts of QkNormParams that forward and backward share; returns V, or 0 on an error
int plan_qk_norm(const char* what, int dtype, int B, int N, int Hq, int Hk, int dh, const void* q, long qb, long qn, long qh,
                 const void* k, long kb, long kn, long kh, const float* table, long rows, int rot, const void* ids, int ids64,
                 long offset, float eps, bool al16, bool al8, int hpt, QkNormParams& p) {
    const int es = dtype == VITK_F32 ? 4 : 2;
    const int V = chunk_elems(es, dh, rot, al16 && aligned(q, qb, qn, qh, es, 16) && aligned(k, kb, kn, kh, es, 16),
                              al8 && aligned(q, qb, qn, qh, es, 8) && aligned(k, kb, kn, kh, es, 8));
    p.table = table;
    p.pos = Pos{ids, ids64, offset, rows};
    p.N = N; p.dh = dh; p.rot = rot; p.eps = eps;
    p.urot = rot / 2 / V;
    p.units = p.urot + (dh - rot + 2 * V - 1) / (2 * V);
    p.lpr_log2 = 0;
    while ((1 << p.lpr_log2) < p.units) ++p.lpr_log2;
    Side* s[2] = {&p.q, &p.k};
    const void* x[2] = {q, k};
    const long st[2][3] = {{qb, qn, qh}, {kb, kn, kh}};
    const int H[2] = {Hq, Hk};
    for (int i = 0; i < 2; ++i) {
        s[i]->x = x[i];
        s[i]->sb = st[i][0]; s[i]->sn = st[i][1]; s[i]->sh = st[i][2];
        s[i]->H = H[i];
        s[i]->hgroups = (H[i] + hpt - 1) / hpt;
        s[i]->groups = (unsigned)B * N * s[i]->hgroups;
    }
    return V;
}
int check_qk_norm(const char* what, int dtype, int B, int N, int Hq, int Hk, int dh, float eps) {
    VITK_CHECK_ARG(dtype == VITK_F32 || dtype == VITK_BF16, "%s: bad dtype %d", what, dtype);
    VITK_CHECK_ARG(B >= 0 && N >= 0 && Hq >= 1 && Hk >= 1, "%s: bad shape B=%d N=%d Hq=%d Hk=%d", what, B, N, Hq, Hk);
    VITK_CHECK_ARG(dh >= 1 && dh <= 128, "%s: head width %d is outside 1 .. 128", what, dh);
    VITK_CHECK_ARG(eps > 0.f, "%s: eps must be positive", what);
    VITK_CHECK_ARG((long)B * N < (1L << 31) && (long)B * N * ((long)Hq + Hk) < (1L << 31),
                   "%s: B * N * (Hq + Hk) = %ld rows are too many for one call", what, (long)B * N * ((long)Hq + Hk));
    return VITK_OK;
}
unsigned side_blocks(long groups, int lpr_log2, unsigned most) {
    const long per = 256 >> lpr_log2;
    const long b = (groups + per - 1) / per;
    if (!most || b <= (long)most) return (unsigned)b;
    const long steps = (b + most - 1) / most;            // every workgroup takes as many steps as the others, or one less
    return (unsigned)((b + steps - 1) / steps);
}

}  // namespace

extern "C" int vitk_rotary_table(int pos_kind, int axes, long rows, const void* positions, int pairs, const double* freqs_host,
                                 double mul, float* table, hipStream_t stream) {
    VITK_CHECK_ARG(pos_kind >= 0 && pos_kind <= 3, "vitk_rotary_table: bad position type %d", pos_kind);
    VITK_CHECK_ARG(axes >= 1 && pairs >= 1 && pairs % axes == 0 && pairs / axes <= 128,
                   "vitk_rotary_table: %d pairs over %d axes (1 .. 128 pairs an axis)", pairs, axes);
    VITK_CHECK_ARG(rows >= 0, "vitk_rotary_table: bad row count");
    if (rows == 0) return VITK_OK;
    VITK_CHECK_ARG(positions && freqs_host && table, "vitk_rotary_table: null pointer");
    Freqs f = {};
    const int per = pairs / axes;
    for (int i = 0; i < per; ++i) f.f[i] = freqs_host[i];
    const long total = rows * pairs;
    const unsigned blocks = (unsigned)((total + 255) / 256 < 65536 ? (total + 255) / 256 : 65536);
#define GO(P) hipLaunchKernelGGL((rotary_table_kernel<P>), dim3(blocks), dim3(256), 0, stream, f, static_cast<const P*>(positions), axes, rows, pairs, per, mul, table)
    switch (pos_kind) {
        case 0: GO(int); break;
        case 1: GO(long long); break;
        case 2: GO(float); break;
        default: GO(double); break;
    }
#undef GO
    VITK_CHECK_LAUNCH("vitk_rotary_table");
    return VITK_OK;
}

extern "C" int vitk_rotary(int dtype, int inverse, int interleaved, int B, int N, int H, int dh, const void* x, long sb, long sn, long sh,
                           const float* table, long table_rows, int rot, const void* pos, int pos64, long offset, void* y,
                           hipStream_t stream) {
    VITK_CHECK_ARG(dtype == VITK_F32 || dtype == VITK_BF16, "vitk_rotary: bad dtype %d", dtype);
    VITK_CHECK_ARG(B >= 0 && N >= 0 && H >= 1 && dh >= 1, "vitk_rotary: bad shape B=%d N=%d H=%d dh=%d", B, N, H, dh);
    if (int e = check_pos("vitk_rotary", table, table_rows, N, rot, dh, pos, offset)) return e;
    if (B == 0 || N == 0) return VITK_OK;
    VITK_CHECK_ARG(x && y, "vitk_rotary: null pointer");
    const int es = dtype == VITK_F32 ? 4 : 2;
    const uintptr_t ya = reinterpret_cast<uintptr_t>(y);
    const int V = chunk_elems(es, dh, rot, aligned(x, sb, sn, sh, es, 16) && ya % 16 == 0, aligned(x, sb, sn, sh, es, 8) && ya % 8 == 0);
    RotaryParams p;
    p.x = x; p.y = y;
    p.sb = sb; p.sn = sn; p.sh = sh;
    p.table = table;
    p.pos = Pos{pos, pos64, offset, table_rows};
    p.N = N; p.H = H; p.dh = dh; p.rot = rot;
    p.urot = rot / 2 / V;
    p.units = p.urot + (dh - rot + 2 * V - 1) / (2 * V);
    p.sgn = inverse ? -1.f : 1.f;
    // four heads a lane, with one read of the turn for them, where that leaves every CU a workgroup or more (32 x 577 tokens x
    // 12 heads of 64: 11.8 us, with one head a lane 14.7); one where the call is small
    const bool wide = H >= 4 && (long)B * N * ((H + 3) / 4) * p.units >= 256L * 256;
    p.hgroups = wide ? (H + 3) / 4 : H;
    const long total = (long)B * N * p.hgroups * p.units;
    VITK_CHECK_ARG(total < (1L << 31) && (long)B * N < (1L << 31), "vitk_rotary: %ld work items are too many for one call", total);
    p.total = (unsigned)total;
    if (es == 2) {
        if (V == 8) launch_rotary<__bf16, 8>(p, interleaved, wide, stream);
        else if (V == 4) launch_rotary<__bf16, 4>(p, interleaved, wide, stream);
        else launch_rotary<__bf16, 1>(p, interleaved, wide, stream);
    } else {
        if (V == 4) launch_rotary<float, 4>(p, interleaved, wide, stream);
        else if (V == 2) launch_rotary<float, 2>(p, interleaved, wide, stream);
        else launch_rotary<float, 1>(p, interleaved, wide, stream);
    }
    VITK_CHECK_LAUNCH("vitk_rotary");
    return VITK_OK;
}

extern "C" int vitk_qk_norm_rotary_fwd(int dtype, int interleaved, int B, int N, int Hq, int Hk, int dh, const void* q, long qb, long qn,
                                       long qh, const void* k, long kb, long kn, long kh, const float* gamma_q,
                                       const float* gamma_k, float eps, const float* table, long table_rows, int rot,
                                       const void* pos, int pos64, long offset, void* yq, void* yk, hipStream_t stream) {
    const char* what = "vitk_qk_norm_rotary_fwd";
    if (int e = check_qk_norm(what, dtype, B, N, Hq, Hk, dh, eps)) return e;
    if (int e = check_pos(what, table, table_rows, N, rot, dh, pos, offset)) return e;
    if (B == 0 || N == 0) return VITK_OK;
    VITK_CHECK_ARG(q && k && yq && yk, "%s: null pointer", what);
    const uintptr_t ya = reinterpret_cast<uintptr_t>(yq) | reinterpret_cast<uintptr_t>(yk);
    QkNormParams p = {};
    const int hpt = large_norm(B, N, Hq + Hk, dh) ? HEADS_FWD : 1;
    const int V = plan_qk_norm(what, dtype, B, N, Hq, Hk, dh, q, qb, qn, qh, k, kb, kn, kh, table, table_rows, rot, pos, pos64, offset, eps,
                               ya % 16 == 0, ya % 8 == 0, hpt, p);
    p.q.gamma = gamma_q; p.k.gamma = gamma_k;
    p.q.y = yq; p.k.y = yk;
    p.q.blocks = side_blocks(p.q.groups, p.lpr_log2, 0);
    p.k.blocks = side_blocks(p.k.groups, p.lpr_log2, 0);
    VITK_CHECK_ARG((long)p.q.blocks + p.k.blocks < (1L << 24), "%s: too many workgroups for one call", what);      // 2^32 threads
    if (dtype == VITK_BF16) {
        if (V == 8) launch_qk_norm<__bf16, 8, false>(p, interleaved, hpt, stream);
        else if (V == 4) launch_qk_norm<__bf16, 4, false>(p, interleaved, hpt, stream);
        else launch_qk_norm<__bf16, 1, false>(p, interleaved, hpt, stream);
    } else {
        if (V == 4) launch_qk_norm<float, 4, false>(p, interleaved, hpt, stream);
        else if (V == 2) launch_qk_norm<float, 2, false>(p, interleaved, hpt, stream);
        else launch_qk_norm<float, 1, false>(p, interleaved, hpt, stream);
    }
    VITK_CHECK_LAUNCH(what);
    return VITK_OK;
}

extern "C" long vitk_qk_norm_rotary_bwd_workspace_bytes(int dh) { return 2L * NORM_BLOCKS * dh * (long)sizeof(float); }

extern "C" int vitk_qk_norm_rotary_bwd(int dtype, int interleaved, int B, int N, int Hq, int Hk, int dh, const void* q, long qb, long qn,
                                       long qh, const void* k, long kb, long kn, long kh, const float* gamma_q,
                                       const float* gamma_k, float eps, const float* table, long table_rows, int rot,
                                       const void* pos, int pos64, long offset, const void* dyq, long gqb, long gqn, long gqh,
                                       const void* dyk, long gkb, long gkn, long gkh, void* dxq, void* dxk, float* dgamma_q,
                                       float* dgamma_k, void* workspace, hipStream_t stream) {
    const char* what = "vitk_qk_norm_rotary_bwd";
    if (int e = check_qk_norm(what, dtype, B, N, Hq, Hk, dh, eps)) return e;
    if (int e = check_pos(what, table, table_rows, N, rot, dh, pos, offset)) return e;
    const bool any_dg = dgamma_q || dgamma_k;
    VITK_CHECK_ARG(!any_dg || workspace, "%s: the gradients of gamma need a workspace", what);
    const bool rows = B > 0 && N > 0;
    QkNormParams p = {};
    if (rows) {
        VITK_CHECK_ARG(q && k && dyq && dyk && dxq && dxk, "%s: null pointer", what);
        const int es = dtype == VITK_F32 ? 4 : 2;
        const uintptr_t ya = reinterpret_cast<uintptr_t>(dxq) | reinterpret_cast<uintptr_t>(dxk);
        const bool al16 = ya % 16 == 0 && aligned(dyq, gqb, gqn, gqh, es, 16) && aligned(dyk, gkb, gkn, gkh, es, 16);
        const bool al8 = ya % 8 == 0 && aligned(dyq, gqb, gqn, gqh, es, 8) && aligned(dyk, gkb, gkn, gkh, es, 8);
        const int hpt = large_norm(B, N, Hq + Hk, dh) ? HEADS_BWD : 1;
        const int V = plan_qk_norm(what, dtype, B, N, Hq, Hk, dh, q, qb, qn, qh, k, kb, kn, kh, table, table_rows, rot, pos, pos64,
                                   offset, eps, al16, al8, hpt, p);
        p.q.gamma = gamma_q; p.k.gamma = gamma_k;
        p.q.dy = dyq; p.q.gb = gqb; p.q.gn = gqn; p.q.gh = gqh;
        p.k.dy = dyk; p.k.gb = gkb; p.k.gn = gkn; p.k.gh = gkh;
        p.q.y = dxq; p.k.y = dxk;
        p.q.blocks = side_blocks(p.q.groups, p.lpr_log2, NORM_BLOCKS);
        p.k.blocks = side_blocks(p.k.groups, p.lpr_log2, NORM_BLOCKS);
        float* ws = static_cast<float*>(workspace);
        p.q.part = dgamma_q ? ws : nullptr;
        p.k.part = dgamma_k ? ws + (long)NORM_BLOCKS * dh : nullptr;
        if (dtype == VITK_BF16) {
            if (V == 8) launch_qk_norm<__bf16, 8, true>(p, interleaved, hpt, stream);
            else if (V == 4) launch_qk_norm<__bf16, 4, true>(p, interleaved, hpt, stream);
            else launch_qk_norm<__bf16, 1, true>(p, interleaved, hpt, stream);
        } else {
            if (V == 4) launch_qk_norm<float, 4, true>(p, interleaved, hpt, stream);
            else if (V == 2) launch_qk_norm<float, 2, true>(p, interleaved, hpt, stream);
            else launch_qk_norm<float, 1, true>(p, interleaved, hpt, stream);
        }
    }
    if (any_dg)      // with no rows the sums are zero, and the kernel below writes that
        hipLaunchKernelGGL(qk_norm_dgamma_kernel, dim3((dh + 15) / 16, 2), dim3(256), 0, stream, p.q.part, p.k.part, p.q.blocks,
                           p.k.blocks, dh, dgamma_q, dgamma_k);
    VITK_CHECK_LAUNCH(what);
    return VITK_OK;
}
