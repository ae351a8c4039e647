// Window attention of one new token a sequence against a ring cache, the append in the same pass; and the fill of the ring
// by whole prompts.
//
// Cache: k, v [B][Hk][C][dh].  Token p of a sequence lives in slot p for p < S (the sinks stay) and S + (p - S) mod (C - S)
// after them; C - S >= w + 1, so the window and the new token are always there.  With window < 0 nothing is overwritten: slot
// p is token p.
//   o = sum_j softmax_j(scale q . k_j) v_j   over j < S and p - w <= j <= p,  p = lengths[b] the new token's own position
//
// The visible part of the cache is read once: that is the bound (2 dh values a key for 4 dh G flops), or the latency of one
// launch where there is little of it.  A key's row is 16-byte chunks on neighbouring lanes, so a wave reads several whole rows
// an instruction; each of those lane groups keeps a running maximum and sum of its own over the keys it meets, and they are
// joined once at the end: no exchange between keys inside the loop.  All of the group's query heads (up to 4 at once) use a
// key while it is in registers.  Where the sequences and heads alone do not fill the card, the keys are dealt to several
// workgroups and a second kernel joins their (maximum, sum, vector) in order.
#include "common.h"

namespace vitk {

struct DecodeParams {
    const void *q, *k, *v;               // q [B][Hq][dh], k / v [B][Hk][dh] with row strides below
    long qb, qh, kb, kh, vb, vh;
    void *kc, *vc;                       // [B][Hk][C][dh]
    const int* lengths;                  // [B]: tokens before the new one; < 0: the sequence takes no part
    void* out;                           // [B][Hq][dh]
    float* part;                         // splits > 1: [B][Hq][splits][2 + dh] (maximum in log2, sum, vector)
    int Hq, Hk, G, dh, C, w, S;
    int splits, gblocks;
    long keys_per_split;
    float sc2;
};

__device__ __forceinline__ float lane_xor(float v, int m) { return __shfl_xor(v, m, 64); }
template <int CTRL> __device__ __forceinline__ float dpp(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
// sum over LPK neighbouring lanes, in every one of them (vector unit up to 16; a shuffle would go through LDS)
template <int LPK> __device__ __forceinline__ float group_sum(float v) {
    if (LPK > 1) v += dpp<0xB1>(v);      // quad_perm [1,0,3,2]
    if (LPK > 2) v += dpp<0x4E>(v);      // quad_perm [2,3,0,1]
    if (LPK > 4) v += dpp<0x141>(v);     // row_half_mirror
    if (LPK > 8) v += dpp<0x140>(v);     // row_mirror
    if (LPK > 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
        v = __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
    }
    return v;
}

template <typename T> struct Row16;                       // 16 bytes of a row as floats
template <> struct Row16<__bf16> { static constexpr int N = 8; };
template <> struct Row16<float> { static constexpr int N = 4; };
template <typename T> __device__ __forceinline__ void unpack16(const u32x4& r, float* f) {
    struct A { T e[Row16<T>::N]; };
    const A a = __builtin_bit_cast(A, r);
#pragma unroll
    for (int i = 0; i < Row16<T>::N; ++i) f[i] = (float)a.e[i];
}

// lane g of the row of 16 lanes, to all of them; g: a constant after unrolling
__device__ __forceinline__ float bcast16(float x, int g) {
    switch (g) {
        case 0: return dpp<0x150>(x);    // row_newbcast:0
        case 1: return dpp<0x151>(x);
        case 2: return dpp<0x152>(x);
        case 3: return dpp<0x153>(x);
        case 4: return dpp<0x154>(x);
        case 5: return dpp<0x155>(x);
        case 6: return dpp<0x156>(x);
        default: return dpp<0x157>(x);
    }
}

// the waves' (maximum, sum, vector) of nh query heads, in order, to out or to the split's place
template <typename T, int GB, int NW, int W>
__device__ __forceinline__ void join_waves(const DecodeParams& p, const float (&sm)[NW][GB][2], const float (&sv)[NW][GB][W], long row0, int nh,
                                           int split, bool lost) {
    for (int x = threadIdx.x; x < nh * p.dh; x += 64 * NW) {
        const int g = x / p.dh, dd = x - g * p.dh;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; ++w) M = fmaxf(M, sm[w][g][0]);
        float L = 0.f, a = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float mw = sm[w][g][0], lw = sm[w][g][1];
            const float f = mw == -INFINITY ? (lw == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(mw - M);
            L += lw * f;
            a += sv[w][g][dd] * f;
        }
        const long row = row0 + g;
        if (p.splits == 1) {
            const float o = lost ? __builtin_nanf("") : (L == 0.f ? 0.f : a / L);
            static_cast<T*>(p.out)[row * p.dh + dd] = (T)o;
        } else {
            float* w = p.part + (row * p.splits + split) * (2 + p.dh);
            if (dd == 0) {
                w[0] = M;
                w[1] = L;
            }
            w[2 + dd] = a;
        }
    }
}

// What sequence b sees, as a list of n tokens: n1 sinks, then lo .. pos.  Slot of entry t: t for the sinks, then a run of the ring
// that starts at `base` and wraps once at most.
struct Seen {
    int n, n1, base, S, R;
    bool lost;                           // a cache without window is full: NaN out, nothing written
};
__device__ __forceinline__ Seen seen_by(const DecodeParams& p, int pos) {
    Seen s;
    s.lost = p.w < 0 && pos >= p.C;
    s.n1 = pos < 0 || s.lost || p.w < 0 ? 0 : (pos < p.S ? pos + 1 : p.S);
    const int lo = p.w < 0 ? 0 : max(p.S, pos - p.w);
    s.n = pos < 0 || s.lost ? 0 : s.n1 + max(0, pos - lo + 1);
    s.R = p.w < 0 ? p.C : p.C - p.S;
    s.S = p.w < 0 ? 0 : p.S;
    s.base = s.n > s.n1 ? (lo - s.S) % s.R : 0;
    return s;
}
__device__ __forceinline__ int seen_slot(const Seen& s, int t) {
    if (t < s.n1) return t;
    const int x = s.base + t - s.n1;
    return s.S + (x >= s.R ? x - s.R : x);
}

template <typename T, int LPK, int GB, int NW, int U>
__global__ __launch_bounds__(64 * NW) void window_decode_kernel(const DecodeParams p) {
    constexpr int E = Row16<T>::N;                        // U: keys in flight a lane group
    constexpr int SLOTS = 64 / LPK, STEP = NW * SLOTS * U;
    __shared__ float sm[NW][GB][2];
    __shared__ float sv[NW][GB][LPK * E];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c = lane % LPK, slot = wave * SLOTS + lane / LPK;
    const int split = blockIdx.x % p.splits;
    const long r1 = blockIdx.x / p.splits;
    const int gb = (int)(r1 % p.gblocks);
    const long bh = r1 / p.gblocks;
    const int hk = (int)(bh % p.Hk);
    const long b = bh / p.Hk;
    const int h0 = hk * p.G + gb * GB, nh = min(GB, p.G - gb * GB);
    const bool act = c * E < p.dh;
    const int d = act ? c * E : 0;

    const Seen sn = seen_by(p, p.lengths[b]);
    const bool lost = sn.lost;
    const int n = sn.n;
    const T* K = static_cast<const T*>(p.kc) + bh * p.C * p.dh;
    const T* V = static_cast<const T*>(p.vc) + bh * p.C * p.dh;
    const T* kn = static_cast<const T*>(p.k) + b * p.kb + (long)hk * p.kh;
    const T* vn = static_cast<const T*>(p.v) + b * p.vb + (long)hk * p.vh;

    float q[GB][E], acc[GB][E], m[GB], l[GB];
#pragma unroll
    for (int g = 0; g < GB; ++g) {
        u32x4 r = {0, 0, 0, 0};
        if (act && g < nh) r = *reinterpret_cast<const u32x4*>(static_cast<const T*>(p.q) + b * p.qb + (long)(h0 + g) * p.qh + d);
        unpack16<T>(r, q[g]);
        m[g] = -INFINITY;
        l[g] = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            q[g][e] *= p.sc2;
            acc[g][e] = 0.f;
        }
    }
    const long t0 = split * p.keys_per_split, t1 = min((long)n, t0 + p.keys_per_split);
    for (long tt = t0; tt < t1; tt += STEP) {
        u32x4 kr[U], vr[U];
        bool ok[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long t = tt + u * (NW * SLOTS) + slot;
            ok[u] = t < t1;
            kr[u] = vr[u] = u32x4{0, 0, 0, 0};
            if (ok[u] && act) {
                const int x = seen_slot(sn, (int)t);
                const bool own = t == n - 1;              // the new token: from the inputs, and into the cache
                kr[u] = *reinterpret_cast<const u32x4*>(own ? kn + d : K + (long)x * p.dh + d);
                vr[u] = *reinterpret_cast<const u32x4*>(own ? vn + d : V + (long)x * p.dh + d);
                if (own && gb == 0) {
                    *reinterpret_cast<u32x4*>(static_cast<T*>(p.kc) + (bh * p.C + x) * p.dh + d) = kr[u];
                    *reinterpret_cast<u32x4*>(static_cast<T*>(p.vc) + (bh * p.C + x) * p.dh + d) = vr[u];
                }
            }
        }
        float s[U][GB];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float f[E];
            unpack16<T>(kr[u], f);
#pragma unroll
            for (int g = 0; g < GB; ++g) {
                float a = 0.f;
#pragma unroll
                for (int e = 0; e < E; ++e) a += q[g][e] * f[e];
                a = group_sum<LPK>(a);
                s[u][g] = ok[u] ? a : -INFINITY;
            }
        }
#pragma unroll
        for (int g = 0; g < GB; ++g) {
            float mn = m[g];
#pragma unroll
            for (int u = 0; u < U; ++u) mn = fmaxf(mn, s[u][g]);
            const float mr = mn == -INFINITY ? 0.f : mn;
            const float al = __builtin_amdgcn_exp2f(m[g] - mr);
            m[g] = mn;
            l[g] *= al;
#pragma unroll
            for (int e = 0; e < E; ++e) acc[g][e] *= al;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                s[u][g] = __builtin_amdgcn_exp2f(s[u][g] - mr);
                l[g] += s[u][g];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float f[E];
            unpack16<T>(vr[u], f);
#pragma unroll
            for (int g = 0; g < GB; ++g)
#pragma unroll
                for (int e = 0; e < E; ++e) acc[g][e] += s[u][g] * f[e];
        }
    }
    // join the wave's lane groups, then the waves
#pragma unroll
    for (int g = 0; g < GB; ++g) {
        float M = m[g];
#pragma unroll
        for (int o = LPK; o < 64; o <<= 1) M = fmaxf(M, lane_xor(M, o));
        const float f = m[g] == -INFINITY ? (l[g] == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(m[g] - M);
        l[g] *= f;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[g][e] *= f;
#pragma unroll
        for (int o = LPK; o < 64; o <<= 1) {
            l[g] += lane_xor(l[g], o);
#pragma unroll
            for (int e = 0; e < E; ++e) acc[g][e] += lane_xor(acc[g][e], o);
        }
        if (lane < LPK) {
#pragma unroll
            for (int e = 0; e < E; ++e) sv[wave][g][lane * E + e] = acc[g][e];
            if (lane == 0) {
                sm[wave][g][0] = M;
                sm[wave][g][1] = l[g];
            }
        }
    }
    __syncthreads();
    join_waves<T, GB, NW, LPK * E>(p, sm, sv, b * p.Hq + h0, nh, split, lost);
}

// bf16 and two query heads or more to a key head: the scores of 16 keys and (up to 16) heads are one chain of 16 x 16 x 32
// MFMA, straight from the cache's rows (a lane holds 16 bytes of key l & 15).  They come out with head l & 15 on the lane and
// keys 4 (l >> 4) .. + 3 in its registers; V is read so that the same 16 lanes hold those 4 keys' rows, and a probability
// reaches the row's lanes by a broadcast within 16 lanes.  On the vector unit the scores took 8 products, 8 conversions and
// 4 exchanges a head and 16 bytes of K: 64 sequences x 4 key heads x 4 x 4100 keys of 128 (447 MB, the caches
// part full) took 222 us in place of 87 (5.1 TB/s, a large copy's rate).  (fp32 takes the vector unit's kernel: full caches of
// that size, 1075 MB, 194 us = 5.5 TB/s, so its bytes bound it there too; bf16 101 us = 5.3.)
typedef __attribute__((ext_vector_type(4))) float f32v4;
template <int LPK, int GB, int NW>
__global__ __launch_bounds__(64 * NW) void window_decode_group_kernel(const DecodeParams p) {
    typedef __bf16 T;
    constexpr int KB = (LPK * 8 + 31) / 32;               // 32-deep K blocks of a row
    constexpr int KPR = 16 / LPK;                         // keys that 16 lanes read at a time
    constexpr int U = 2;                                  // tiles of 16 keys in flight a wave
    constexpr int STEP = NW * 16 * U;
    __shared__ float sm[NW][GB][2];
    __shared__ float sv[NW][GB][LPK * 8];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = lane >> 4, i = lane & 15;             // 16 lanes: their 4 keys; key (K) / head (scores) / chunk (V)
    const int c = i % LPK, sub = i / LPK;
    const int split = blockIdx.x % p.splits;
    const long r1 = blockIdx.x / p.splits;
    const int gb = (int)(r1 % p.gblocks);
    const long bh = r1 / p.gblocks;
    const int hk = (int)(bh % p.Hk);
    const long b = bh / p.Hk;
    const int h0 = hk * p.G + gb * GB, nh = min(GB, p.G - gb * GB);
    const bool act = c * 8 < p.dh;

    const Seen sn = seen_by(p, p.lengths[b]);
    const T* K = static_cast<const T*>(p.kc) + bh * p.C * p.dh;
    const T* V = static_cast<const T*>(p.vc) + bh * p.C * p.dh;
    const T* kn = static_cast<const T*>(p.k) + b * p.kb + (long)hk * p.kh;
    const T* vn = static_cast<const T*>(p.v) + b * p.vb + (long)hk * p.vh;
    bf16x8 qf[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
        const int d = 32 * kb + 8 * row;
        u32x4 r = {0, 0, 0, 0};
        if (i < nh && d < p.dh) r = *reinterpret_cast<const u32x4*>(static_cast<const T*>(p.q) + b * p.qb + (long)(h0 + i) * p.qh + d);
        qf[kb] = __builtin_bit_cast(bf16x8, r);
    }
    float acc[GB][8], m = -INFINITY, l = 0.f;             // m, l: head i's, over this row of lanes' keys
#pragma unroll
    for (int g = 0; g < GB; ++g)
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[g][e] = 0.f;

    const long t0 = split * p.keys_per_split, t1 = min((long)sn.n, t0 + p.keys_per_split);
    for (long tt = t0 + 16 * U * wave; tt < t1; tt += STEP) {     // the same for the whole wave
        u32x4 kr[U][KB], vr[U][4 / KPR];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long t = tt + 16 * u + i;
            const bool own = t == sn.n - 1;               // the new token: from the inputs, and into the cache
            const long x = t < t1 ? seen_slot(sn, (int)t) : 0;
            const T* from = own ? kn : K + x * p.dh;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                const int d = 32 * kb + 8 * row;
                kr[u][kb] = u32x4{0, 0, 0, 0};
                if (t < t1 && d < p.dh) {
                    kr[u][kb] = *reinterpret_cast<const u32x4*>(from + d);
                    if (own && gb == 0) *reinterpret_cast<u32x4*>(static_cast<T*>(p.kc) + (bh * p.C + x) * p.dh + d) = kr[u][kb];
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < 4 / KPR; ++j) {
                const long t = tt + 16 * u + 4 * row + KPR * j + sub;
                vr[u][j] = u32x4{0, 0, 0, 0};
                if (t < t1 && act) {
                    const bool own = t == sn.n - 1;
                    const long x = seen_slot(sn, (int)t);
                    vr[u][j] = *reinterpret_cast<const u32x4*>((own ? vn : V + x * p.dh) + 8 * c);
                    if (own && gb == 0) *reinterpret_cast<u32x4*>(static_cast<T*>(p.vc) + (bh * p.C + x) * p.dh + 8 * c) = vr[u][j];
                }
            }
        f32v4 s[U];
        float mt = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            s[u] = f32v4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
                s[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kr[u][kb]), qf[kb], s[u], 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[u][r] = tt + 16 * u + 4 * row + r < t1 ? s[u][r] * p.sc2 : -INFINITY;
                mt = fmaxf(mt, s[u][r]);
            }
        }
        if (__any(mt > m + 8.f)) {                        // the reference point moves with 2^8, as in the prefill
            const float mn = fmaxf(m, mt);
            const float al = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= al;
#pragma unroll
            for (int g = 0; g < GB; ++g) {
                const float ag = bcast16(al, g);
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[g][e] *= ag;
            }
        }
        const float mr = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[u][r] = __builtin_amdgcn_exp2f(s[u][r] - mr);
                l += s[u][r];
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < 4 / KPR; ++j) {
                float f[8];
                unpack16<T>(vr[u][j], f);
#pragma unroll
                for (int g = 0; g < GB; ++g) {
                    float pk[KPR], pg;                    // the broadcasts need all 16 lanes: no choice around them
#pragma unroll
                    for (int k = 0; k < KPR; ++k) pk[k] = bcast16(s[u][KPR * j + k], g);
                    pg = pk[0];
#pragma unroll
                    for (int k = 1; k < KPR; ++k) pg = sub == k ? pk[k] : pg;
#pragma unroll
                    for (int e = 0; e < 8; ++e) acc[g][e] += pg * f[e];
                }
            }
    }
    // join the wave's 4 rows of lanes (and the keys that shared one), then the waves
    float M = m;
    M = fmaxf(M, lane_xor(M, 16));
    M = fmaxf(M, lane_xor(M, 32));
    const float f = m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(m - M);
    l *= f;
    l += lane_xor(l, 16);
    l += lane_xor(l, 32);
    if (lane < nh) {
        sm[wave][lane][0] = M;
        sm[wave][lane][1] = l;
    }
#pragma unroll
    for (int g = 0; g < GB; ++g) {
        const float fg = bcast16(f, g);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            acc[g][e] *= fg;
#pragma unroll
            for (int o = LPK; o < 64; o <<= 1) acc[g][e] += lane_xor(acc[g][e], o);
            if (lane < LPK) sv[wave][g][lane * 8 + e] = acc[g][e];
        }
    }
    __syncthreads();
    join_waves<T, GB, NW, LPK * 8>(p, sm, sv, b * p.Hq + h0, nh, split, sn.lost);
}

// joins the splits of one (sequence, query head), in order
template <typename T>
__global__ __launch_bounds__(128) void window_decode_join_kernel(const DecodeParams p) {
    const long row = blockIdx.x;
    const int d = threadIdx.x;
    if (d >= p.dh) return;
    const float* w = p.part + row * p.splits * (2 + p.dh);
    float M = -INFINITY, L = 0.f, a = 0.f;
    for (int s = 0; s < p.splits; ++s) M = fmaxf(M, w[(long)s * (2 + p.dh)]);
    for (int s = 0; s < p.splits; ++s) {
        const float* x = w + (long)s * (2 + p.dh);
        const float f = x[0] == -INFINITY ? (x[1] == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(x[0] - M);
        L += x[1] * f;
        a += x[2 + d] * f;
    }
    const bool lost = p.w < 0 && p.lengths[row / p.Hq] >= p.C;
    static_cast<T*>(p.out)[row * p.dh + d] = (T)(lost ? __builtin_nanf("") : (L == 0.f ? 0.f : a / L));
}

// Every slot takes the last token of the prompt that belongs in it; slots that the prompt does not reach are left alone.
struct FillParams {
    const void *k, *v;                   // element (b, n, h, d) at b*sb + n*sn + h*sh + d
    long kb, kn, kh, vb, vn, vh;
    void *kc, *vc;
    const int* lengths;                  // [B] or NULL: N tokens
    int N, Hk, C, S, row_chunks, dh;
    long total;                          // B * Hk * C * chunks of 16 bytes a row
};
template <typename T>
__global__ __launch_bounds__(256) void window_cache_fill_kernel(const FillParams p) {
    constexpr int E = Row16<T>::N;
    for (long id = (long)blockIdx.x * 256 + threadIdx.x; id < p.total; id += (long)gridDim.x * 256) {
        const long r = id / p.row_chunks;
        const int d = (int)(id - r * p.row_chunks) * E;
        const long bh = r / p.C;
        const int c = (int)(r - bh * p.C);
        const long b = bh / p.Hk;
        const int h = (int)(bh - b * p.Hk);
        const int n = p.lengths ? max(0, min(p.lengths[b], p.N)) : p.N;
        const int R = p.C - p.S;
        int t = c;                       // the last token before n that has this slot
        if (c >= p.S && n > c) t = c + (n - 1 - c) / R * R;
        if (t >= n) continue;
        *reinterpret_cast<u32x4*>(static_cast<T*>(p.kc) + r * p.dh + d) =
            *reinterpret_cast<const u32x4*>(static_cast<const T*>(p.k) + b * p.kb + (long)t * p.kn + (long)h * p.kh + d);
        *reinterpret_cast<u32x4*>(static_cast<T*>(p.vc) + r * p.dh + d) =
            *reinterpret_cast<const u32x4*>(static_cast<const T*>(p.v) + b * p.vb + (long)t * p.vn + (long)h * p.vh + d);
    }
}

}  // namespace vitk

using namespace vitk;

namespace {

int check_cache(const char* what, int dtype, int B, int Hq, int Hk, int dh, int C, int window, int sinks) {
    VITK_CHECK_ARG(dtype == VITK_F32 || dtype == VITK_BF16, "%s: bad dtype %d", what, dtype);
    VITK_CHECK_ARG(B >= 0 && Hq >= 1 && Hk >= 1 && Hq % Hk == 0, "%s: bad shape B=%d Hq=%d Hk=%d", what, B, Hq, Hk);
    VITK_CHECK_ARG(dh >= 8 && dh <= 128 && dh % 8 == 0, "%s: head width %d must be a multiple of 8 up to 128", what, dh);
    VITK_CHECK_ARG(C >= 1 && C < (1 << 28) && sinks >= 0, "%s: bad cache of %d slots with %d sinks", what, C, sinks);
    VITK_CHECK_ARG(window < 0 || (long)C >= (long)sinks + window + 1, "%s: %d slots cannot hold %d sinks, a window of %d and the new token",
                   what, C, sinks, window);
    return VITK_OK;
}
bool al16(const void* p, int es, long a, long b = 0, long c = 0) {
    return p && (reinterpret_cast<uintptr_t>(p) & 15) == 0 && a * es % 16 == 0 && b * es % 16 == 0 && c * es % 16 == 0;
}

struct DecodePlan { int splits, gb, gblocks, nw; long per; };
// Waves a workgroup and workgroups a row (sequence, key head, up to 4 query heads).  Up to 256 KiB of keys and values a row is
// one workgroup's work, of 16 waves where there are few rows: a second kernel costs more than it saves.  Beyond, keys are
// dealt to so many workgroups that every CU has 8 waves or more (256 rows of 4100 keys of 128, bf16, groups of 4: 88 us with
// one workgroup of 8 waves a row, 96 with two and the join, 129 with 16 waves, whose registers spill).
DecodePlan decode_plan(int B, int Hq, int Hk, int dh, int C, int w, int S, int es) {
    DecodePlan d;
    const int G = Hq / Hk;
    const bool group = es == 2 && G > 1;
    d.gb = G == 1 ? 1 : (G == 2 ? 2 : 4);
    d.gblocks = (G + d.gb - 1) / d.gb;
    const long most = w < 0 ? C : (long)S + w + 1;
    const long rows = (long)B * Hk * d.gblocks, bytes = most * dh * es * 2;
    const int few = group ? 8 : 16;
    long splits = 1;
    d.nw = rows < 512 ? few : 4;
    if (rows < 192 && bytes > 256 * 1024) {
        d.nw = group ? 8 : 4;
        splits = (2048 / d.nw + rows - 1) / rows;
        const long cap = (bytes + 64 * 1024 - 1) / (64 * 1024);
        if (splits > cap) splits = cap;
        if (splits > 64) splits = 64;
    }
    d.splits = (int)splits;
    d.per = (most + splits - 1) / splits;
    return d;
}

template <typename T, int LPK, int GB> void launch_decode(const DecodeParams& p, int nw, long blocks, hipStream_t st) {
    if (nw == 4) hipLaunchKernelGGL((window_decode_kernel<T, LPK, GB, 4, 4>), dim3((unsigned)blocks), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((window_decode_kernel<T, LPK, GB, 16, 4>), dim3((unsigned)blocks), dim3(1024), 0, st, p);
}
template <int LPK, int GB> void launch_group(const DecodeParams& p, int nw, long blocks, hipStream_t st) {
    if (nw == 4) hipLaunchKernelGGL((window_decode_group_kernel<LPK, GB, 4>), dim3((unsigned)blocks), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((window_decode_group_kernel<LPK, GB, 8>), dim3((unsigned)blocks), dim3(512), 0, st, p);
}
template <typename T, int LPK> void decode_heads(const DecodeParams& p, const DecodePlan& d, long blocks, hipStream_t st) {
    if constexpr (sizeof(T) == 2) {
        if (d.gb == 1) launch_decode<T, LPK, 1>(p, d.nw, blocks, st);
        else if (d.gb == 2) launch_group<LPK, 2>(p, d.nw, blocks, st);
        else launch_group<LPK, 4>(p, d.nw, blocks, st);
    } else {
        if (d.gb == 1) launch_decode<T, LPK, 1>(p, d.nw, blocks, st);
        else if (d.gb == 2) launch_decode<T, LPK, 2>(p, d.nw, blocks, st);
        else launch_decode<T, LPK, 4>(p, d.nw, blocks, st);
    }
}

}  // namespace

extern "C" long vitk_window_decode_workspace_bytes(int dtype, int B, int Hq, int Hk, int dh, int C, int window, int sinks) {
    if (B <= 0 || Hq <= 0 || Hk <= 0 || Hq % Hk || dh <= 0 || C <= 0 || sinks < 0) return 0;
    const DecodePlan d = decode_plan(B, Hq, Hk, dh, C, window, window < 0 ? 0 : sinks, dtype == VITK_F32 ? 4 : 2);
    return d.splits == 1 ? 0 : (long)B * Hq * d.splits * (2 + dh) * 4;
}

extern "C" int vitk_window_decode(int dtype, int B, int Hq, int Hk, int dh, const void* q, long qb, long qh, const void* k, long kb,
                                  long kh, const void* v, long vb, long vh, void* k_cache, void* v_cache, int C, const int* lengths,
                                  float scale, int window, int sinks, void* out, void* workspace, hipStream_t stream) {
    const char* what = "vitk_window_decode";
    if (int e = check_cache(what, dtype, B, Hq, Hk, dh, C, window, sinks)) return e;
    VITK_CHECK_ARG(scale > 0.f && scale < INFINITY, "%s: the scale must be positive and finite", what);
    if (B == 0) return VITK_OK;
    const int es = dtype == VITK_F32 ? 4 : 2;
    VITK_CHECK_ARG(al16(q, es, qb, qh) && al16(k, es, kb, kh) && al16(v, es, vb, vh) && al16(k_cache, es, 0) && al16(v_cache, es, 0) &&
                   out && lengths, "%s: q, k, v and the caches must be 16-byte aligned, their strides too", what);
    DecodeParams p = {};
    p.q = q; p.k = k; p.v = v;
    p.qb = qb; p.qh = qh; p.kb = kb; p.kh = kh; p.vb = vb; p.vh = vh;
    p.kc = k_cache; p.vc = v_cache;
    p.lengths = lengths;
    p.out = out;
    p.part = static_cast<float*>(workspace);
    p.Hq = Hq; p.Hk = Hk; p.G = Hq / Hk; p.dh = dh; p.C = C;
    p.w = window < 0 ? -1 : window;
    p.S = window < 0 ? 0 : sinks;
    p.sc2 = scale * 1.4426950408889634f;
    const DecodePlan d = decode_plan(B, Hq, Hk, dh, C, p.w, p.S, es);
    p.splits = d.splits; p.gblocks = d.gblocks; p.keys_per_split = d.per;
    VITK_CHECK_ARG(d.splits == 1 || workspace, "%s: this shape needs a workspace", what);
    const long blocks = (long)B * Hk * d.gblocks * d.splits;
    VITK_CHECK_ARG(blocks * d.nw * 64 < (1L << 32) && (long)B * Hq * 128 < (1L << 32), "%s: too many workgroups for one call", what);
    const int chunks = dh * es / 16;                      // lanes a key's row takes, up to a power of two
    if (dtype == VITK_BF16) {
        if (chunks <= 4) decode_heads<__bf16, 4>(p, d, blocks, stream);
        else if (chunks <= 8) decode_heads<__bf16, 8>(p, d, blocks, stream);
        else decode_heads<__bf16, 16>(p, d, blocks, stream);
        if (d.splits > 1) hipLaunchKernelGGL((window_decode_join_kernel<__bf16>), dim3((unsigned)((long)B * Hq)), dim3(128), 0, stream, p);
    } else {
        if (chunks <= 4) decode_heads<float, 4>(p, d, blocks, stream);
        else if (chunks <= 8) decode_heads<float, 8>(p, d, blocks, stream);
        else if (chunks <= 16) decode_heads<float, 16>(p, d, blocks, stream);
        else decode_heads<float, 32>(p, d, blocks, stream);
        if (d.splits > 1) hipLaunchKernelGGL((window_decode_join_kernel<float>), dim3((unsigned)((long)B * Hq)), dim3(128), 0, stream, p);
    }
    VITK_CHECK_LAUNCH(what);
    return VITK_OK;
}

extern "C" int vitk_window_cache_fill(int dtype, int B, int N, int Hk, int dh, const void* k, long kb, long kn, long kh, const void* v,
                                      long vb, long vn, long vh, const int* lengths, void* k_cache, void* v_cache, int C, int sinks,
                                      hipStream_t stream) {
    const char* what = "vitk_window_cache_fill";
    if (int e = check_cache(what, dtype, B, Hk, Hk, dh, C, -1, sinks)) return e;
    VITK_CHECK_ARG(N >= 0 && C > sinks, "%s: bad sizes N=%d C=%d sinks=%d", what, N, C, sinks);
    if (B == 0 || N == 0) return VITK_OK;
    const int es = dtype == VITK_F32 ? 4 : 2;
    VITK_CHECK_ARG(al16(k, es, kb, kn, kh) && al16(v, es, vb, vn, vh) && al16(k_cache, es, 0) && al16(v_cache, es, 0),
                   "%s: k, v and the caches must be 16-byte aligned, their strides too", what);
    FillParams p = {};
    p.k = k; p.v = v;
    p.kb = kb; p.kn = kn; p.kh = kh; p.vb = vb; p.vn = vn; p.vh = vh;
    p.kc = k_cache; p.vc = v_cache;
    p.lengths = lengths;
    p.N = N; p.Hk = Hk; p.C = C; p.S = sinks; p.dh = dh;
    p.row_chunks = dh * es / 16;
    p.total = (long)B * Hk * C * p.row_chunks;
    const long blocks = (p.total + 255) / 256;
    const unsigned grid = (unsigned)(blocks < 16384 ? blocks : 16384);
    if (dtype == VITK_BF16) hipLaunchKernelGGL((window_cache_fill_kernel<__bf16>), dim3(grid), dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((window_cache_fill_kernel<float>), dim3(grid), dim3(256), 0, stream, p);
    VITK_CHECK_LAUNCH(what);
    return VITK_OK;
}
