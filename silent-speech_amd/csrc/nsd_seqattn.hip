// Attention of whole sequences (gfx950), for training through the AR head's frozen layers, for prompts, for scored
// candidates, and for beam steps over long shared prefixes:
//   nsd_attn_fwd     O = softmax(scale Q K^T + mask) V and the log-sums L of its rows
//   nsd_attn_bwd     the gradients of Q, K and V, with the probabilities recomputed from L
//   nsd_attn_prefix  the softmax state of a beam's hypotheses over keys that they share
// One formulation serves the three.  The G = heads / kv_heads query heads of a kv head read the same keys, so the rows
// of a (batch, kv head) pair are the R = Lq * G pairs rho = i * G + g of token and head.  A wave owns 32 columns of a
// transposed score tile S^T = K Q^T (v_mfma_f32_32x32x16_bf16, for fp32 v_mfma_f32_32x32x2_f32): a lane then holds, for
// ONE query row, 16 of 32 keys, so maxima and sums of a row are taken in registers with one exchange between the lane
// halves, and the probabilities already lie as the B operand of O^T = V^T P^T - slot j of lane half h is key
// 8 (j / 4) + 4 h + j % 4 of 16, and the V^T operand is read from LDS in that same order of keys (ds_read_b64_tr_b16
// transposes the row-major tile on the way).  Scores, probabilities and sums are fp32; probabilities and their
// gradients are rounded to bf16 only where they enter a bf16 product.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "nsd_device.h"
#include "nsd_elem.h"

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// Eight values of a lane along the contracted axis: the operand of sixteen contracted elements (two lane halves).
template <class T> struct Frag;
template <> struct Frag<BF16> { bf16x8 v; };
template <> struct Frag<float> { float v[8]; };

NSD_D void mma(f32x16 &c, const Frag<BF16> &a, const Frag<BF16> &b)
{
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, b.v, c, 0, 0, 0);
}
NSD_D void mma(f32x16 &c, const Frag<float> &a, const Frag<float> &b)
{
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[j], b.v[j], c, 0, 0, 0);
}

// registers 8c .. 8c+7 of an accumulator as the operand of its rows 16c .. 16c+15
NSD_D Frag<BF16> acc_frag(const f32x16 &s, int c, BF16)
{
    Frag<BF16> f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const f32x2 p = {s[8 * c + 2 * j], s[8 * c + 2 * j + 1]};
        const bf16x2 r = __builtin_convertvector(p, bf16x2);
        f.v[2 * j] = r[0];
        f.v[2 * j + 1] = r[1];
    }
    return f;
}
NSD_D Frag<float> acc_frag(const f32x16 &s, int c, float)
{
    Frag<float> f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f.v[j] = s[8 * c + j];
    return f;
}

NSD_D float half_max(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
NSD_D float half_sum(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
NSD_D float exp2_hw(float v) { return __builtin_amdgcn_exp2f(v); }

// A tile of rows in LDS, DP elements each, in 16-byte pieces.  Piece p of row r lies at p ^ sw(r): eight lanes that
// read the same piece of eight rows (the operand reads along a row) and sixteen lanes that read 32 bytes of four rows
// (the transposing reads) then touch every bank once.
template <class T, int DP> struct Tile {
    static constexpr int RB = DP * (int)sizeof(T);              // bytes of a row
    static constexpr int PR = RB / 16;                          // pieces of a row
    static constexpr bool B16 = sizeof(T) == 2;
    NSD_D static int sw(int row) { return !B16 ? row & 7 : DP == 128 ? (row & 7) << 1 : (row >> 1 & 3) << 1; }
    NSD_D static int at(int row, int piece) { return row * RB + ((piece ^ sw(row)) << 4); }

    // elements 16 kc + 8 h .. + 7 of row `row` (h = lane half)
    NSD_D static Frag<T> row_frag(const char *s, int row, int kc, int h)
    {
        Frag<T> f;
        if constexpr (B16) {
            f.v = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4 *>(s + at(row, 2 * kc + h)));
        } else {
            const float4 x = *reinterpret_cast<const float4 *>(s + at(row, 4 * kc + 2 * h));
            const float4 y = *reinterpret_cast<const float4 *>(s + at(row, 4 * kc + 2 * h + 1));
            f.v[0] = x.x; f.v[1] = x.y; f.v[2] = x.z; f.v[3] = x.w;
            f.v[4] = y.x; f.v[5] = y.y; f.v[6] = y.z; f.v[7] = y.w;
        }
        return f;
    }
    // column 32 dt + (lane & 31) of rows r0 + 4 h + 0..3 and r0 + 8 + 4 h + 0..3 (r0 a multiple of 16)
    NSD_D static Frag<T> col_frag(const char *s, int r0, int dt, int lane)
    {
        Frag<T> f;
        const int h = lane >> 5;
        if constexpr (B16) {
            // sixteen lanes hand in 32 bytes of four rows and get a column of sixteen each
            const int row = r0 + 4 * h + (lane >> 2 & 3);
            const char *p = s + at(row, 4 * dt + 2 * (lane >> 4 & 1) + (lane >> 1 & 1)) + 8 * (lane & 1);
            typedef __attribute__((address_space(3))) s16x4 lds4;
            const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)p);
            const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)(p + 8 * RB));
            f.v = __builtin_bit_cast(bf16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            const int d = 32 * dt + (lane & 31);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int row = r0 + 8 * (j >> 2) + 4 * h + (j & 3);
                f.v[j] = *reinterpret_cast<const float *>(s + at(row, d >> 2) + 4 * (d & 3));
            }
        }
        return f;
    }
};

// The same eight elements straight from a row in memory; zeros past the row's end or for no row.
NSD_D Frag<BF16> mem_frag(const BF16 *row, int d0, int D, bool ok)
{
    uint4 x = make_uint4(0, 0, 0, 0);
    if (ok && d0 < D) x = *reinterpret_cast<const uint4 *>(row + d0);
    Frag<BF16> f;
    f.v = __builtin_bit_cast(bf16x8, x);
    return f;
}
NSD_D Frag<float> mem_frag(const float *row, int d0, int D, bool ok)
{
    float4 x = make_float4(0, 0, 0, 0), y = x;
    if (ok && d0 < D) {
        x = *reinterpret_cast<const float4 *>(row + d0);
        y = *reinterpret_cast<const float4 *>(row + d0 + 4);
    }
    return Frag<float>{{x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w}};
}

// sum over a lane's eight products
NSD_D float frag_dot(const Frag<BF16> &a, const Frag<BF16> &b, float s)
{
#pragma unroll
    for (int j = 0; j < 8; ++j) s = __builtin_fmaf((float)a.v[j], (float)b.v[j], s);
    return s;
}
NSD_D float frag_dot(const Frag<float> &a, const Frag<float> &b, float s)
{
#pragma unroll
    for (int j = 0; j < 8; ++j) s = __builtin_fmaf(a.v[j], b.v[j], s);
    return s;
}

// four consecutive elements of a row, rounded to the element type
NSD_D void store4(float *p, float a, float b, float c, float d) { *reinterpret_cast<float4 *>(p) = make_float4(a, b, c, d); }
NSD_D void store4(BF16 *p, float a, float b, float c, float d)
{
    const f32x2 x = {a, b}, y = {c, d};
    const uint32_t u = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf16x2));
    const uint32_t w = __builtin_bit_cast(uint32_t, __builtin_convertvector(y, bf16x2));
    *reinterpret_cast<uint2 *>(p) = make_uint2(u, w);
}

// ---------------------------------------------------------------------
// arguments.  Strides count elements; rows rho = i * G + g of a (z, kv head) pair, R = Lq * G of them.
// ---------------------------------------------------------------------
struct SeqArgs {
    const void *q, *k, *v;
    int64_t q_sz, q_st, q_sh, k_sz, k_st, k_sh, v_sz, v_st, v_sh;
    const uint8_t *mask;                   // [Z, Lk] or null: keys that rows may see
    const int32_t *lens;                   // [Z] or null: keys that there are, at most Lk
    int Z, KVH, G, Lq, Lk, D, R, causal;
    uint32_t g_magic;                      // rho / G = rho * g_magic >> 32
    float scale2;                          // scale * log2(e): scores are exponents of two
    // forward
    void *out;                             // [Z, Lq, heads, D]
    float *lse;                            // [Z, KVH, R], natural logarithm
    float *po, *pm, *pl;                   // state [splits][Z * Lq * heads] (sum of weighted values, maximum, sum)
    const float *in_o, *in_m, *in_l;       // a state to continue, or null
    int splits, split_tiles;
    // backward
    const void *dout;                      // [Z, Lq, heads, D]
    float *delta;                          // [Z, KVH, R]
    void *dq, *dk, *dv;                    // contiguous like q, k, v
    float scale;
};

NSD_D int div_g(int rho, uint32_t magic, int G) { return G == 1 ? rho : (int)(((uint64_t)(uint32_t)rho * magic) >> 32); }

// the 64 (or fewer) keys from j0 on that exist and are not masked, as a word that every lane has
NSD_D uint64_t key_word(const SeqArgs &a, const uint8_t *mask, int j0, int n_keys)
{
    const int j = j0 + (int)(threadIdx.x & 63);
    bool ok = j < n_keys;
    if (mask && ok) ok = mask[j] != 0;
    return __ballot(ok);
}

// One tile of ROWS rows on its way from memory to LDS, 256 threads: U pieces of 16 bytes for each.
template <class T, int DP, int ROWS> struct Stage {
    static constexpr int PR = Tile<T, DP>::PR, U = ROWS * PR / 256, EP = 16 / (int)sizeof(T);
    uint4 x[U];
    // rows row0 .. of a matrix at `base` with `stride` elements between rows; row r is there if ok(r)
    template <class F> NSD_D void load(const T *base, int64_t stride, int D, F ok)
    {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = (int)threadIdx.x + 256 * u, r = i / PR, p = i % PR;
            x[u] = make_uint4(0, 0, 0, 0);
            if (p * EP < D && ok(r)) x[u] = *reinterpret_cast<const uint4 *>(base + r * stride + p * EP);
        }
    }
    NSD_D void put(char *s) const
    {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = (int)threadIdx.x + 256 * u;
            *reinterpret_cast<uint4 *>(s + Tile<T, DP>::at(i / PR, i % PR)) = x[u];
        }
    }
};

// ---------------------------------------------------------------------
// forward.  A workgroup of four waves: WM of them along the rows (32 each), WN = 4 / WM along the keys (KW of a tile's
// BN = KW * WN each; their states meet at the end).  grid.x = row tile, (z, kv head), split.
// ---------------------------------------------------------------------
template <class T, int DP, int WM, int KW, int NBUF, bool STATE>
__global__ void __launch_bounds__(256)
nsd_attn_fwd_kernel(SeqArgs a)
{
    constexpr int WN = 4 / WM, BM = 32 * WM, BN = KW * WN, NK = KW / 32, DT = DP / 32, KC = DP / 16;
    constexpr int NW = BN > 64 ? BN / 64 : 1;                   // key words of a tile
    using TL = Tile<T, DP>;
    constexpr int TB = BN * TL::RB;                             // bytes of the keys of a tile
    constexpr int JOIN = WN > 1 ? WN * WM * 32 * (DP + 2) * 4 : 0;
    constexpr int SMEM = 2 * NBUF * TB > JOIN ? 2 * NBUF * TB : JOIN;
    __shared__ __align__(16) char smem[SMEM];

    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, c32 = lane & 31;
    const int wm = w % WM, wn = w / WM;
    const int rtiles = (a.R + BM - 1) / BM;
    int bid = blockIdx.x;
    const int split = bid % a.splits;
    bid /= a.splits;
    // later rows of a causal mask see more keys: their tiles start first
    const int rt = rtiles - 1 - bid % rtiles;
    bid /= rtiles;
    const int kvh = bid % a.KVH, z = bid / a.KVH;
    const int n_keys = a.lens ? min(max(a.lens[z], 0), a.Lk) : a.Lk;
    const uint8_t *mask = a.mask ? a.mask + (size_t)z * a.Lk : nullptr;

    const int r0 = rt * BM, rho = r0 + wm * 32 + c32;
    const bool row_ok = rho < a.R;
    const int off = a.Lk - a.Lq;
    const int i_row = div_g(row_ok ? rho : a.R - 1, a.g_magic, a.G);
    const int head = kvh * a.G + ((row_ok ? rho : a.R - 1) - i_row * a.G);
    const int last = a.causal ? i_row + off : a.Lk;             // this row sees keys j <= last
    int kend = n_keys;
    if (a.causal) kend = min(kend, div_g(min(r0 + BM, a.R) - 1, a.g_magic, a.G) + off + 1);
    const int t_end = min((split + 1) * a.split_tiles, kend > 0 ? (kend + BN - 1) / BN : 0);
    int t = split * a.split_tiles;

    const T *kb = static_cast<const T *>(a.k) + z * a.k_sz + kvh * a.k_sh;
    const T *vb = static_cast<const T *>(a.v) + z * a.v_sz + kvh * a.v_sh;
    Frag<T> qf[KC];
    {
        const T *qp = static_cast<const T *>(a.q) + z * a.q_sz + i_row * a.q_st + head * a.q_sh;
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) qf[kc] = mem_frag(qp, 16 * kc + 8 * h, a.D, row_ok);
    }
    const size_t row = ((size_t)z * a.Lq + i_row) * (a.KVH * a.G) + head;       // of out and of the states
    float m = -__builtin_inff(), l = 0.0f;
    f32x16 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[dt][e] = 0.0f;
    if constexpr (STATE) {
        if (a.in_o && split == 0 && wn == 0 && row_ok) {
            m = a.in_m[row] * LOG2E;
            l = h == 0 ? a.in_l[row] : 0.0f;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const int d = 32 * dt + 8 * b + 4 * h;
                    if (d < a.D) {
                        const float4 x = *reinterpret_cast<const float4 *>(a.in_o + row * a.D + d);
                        o[dt][4 * b] = x.x; o[dt][4 * b + 1] = x.y; o[dt][4 * b + 2] = x.z; o[dt][4 * b + 3] = x.w;
                    }
                }
        }
    }

    Stage<T, DP, BN> ks, vs;
    uint64_t word[NW], next[NW];
    auto fetch = [&](int tile) {
        const int j0 = tile * BN;
#pragma unroll
        for (int i = 0; i < NW; ++i) next[i] = key_word(a, mask, j0 + 64 * i, n_keys);
        // rows that no query may see are zeros: what lies there takes no part, not even as 0 * NaN
        auto ok = [&](int r) { return (bool)(next[r >> 6 < NW ? r >> 6 : 0] >> (r & 63) & 1); };
        ks.load(kb + (int64_t)j0 * a.k_st, a.k_st, a.D, ok);
        vs.load(vb + (int64_t)j0 * a.v_st, a.v_st, a.D, ok);
    };
    if (t < t_end) fetch(t);
    for (int buf = 0; t < t_end; ++t, buf = (buf + 1) % NBUF) {
        char *sk = smem + buf * 2 * TB, *sv = sk + TB;
        if (NBUF == 1) __syncthreads();
        ks.put(sk);
        vs.put(sv);
#pragma unroll
        for (int i = 0; i < NW; ++i) word[i] = next[i];
        if (t + 1 < t_end) fetch(t + 1);
        __syncthreads();

        // scores of this wave's KW keys
        f32x16 s[NK];
#pragma unroll
        for (int n = 0; n < NK; ++n) {
#pragma unroll
            for (int e = 0; e < 16; ++e) s[n][e] = 0.0f;
#pragma unroll
            for (int kc = 0; kc < KC; ++kc) mma(s[n], TL::row_frag(sk, wn * KW + 32 * n + c32, kc, h), qf[kc]);
        }
        // the keys that this lane's row sees, of the wave's part of the tile
        const int kw0 = wn * KW;
        uint64_t vis = word[NW > 1 ? kw0 >> 6 : 0] >> (kw0 & 63);
        const int n_vis = last + 1 - (t * BN + kw0);
        vis = n_vis <= 0 ? 0 : n_vis < 64 ? vis & ((1ull << n_vis) - 1) : vis;
        const uint64_t all = KW == 64 ? ~0ull : (1ull << (KW & 63)) - 1;
        if (__ballot((vis & all) != all) != 0) {
#pragma unroll
            for (int n = 0; n < NK; ++n) {
                const uint32_t bits = (uint32_t)(vis >> (32 * n)) >> (4 * h);
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    s[n][e] = bits >> (8 * (e >> 2) + (e & 3)) & 1 ? s[n][e] : -__builtin_inff();
            }
        }
        float mx = s[0][0];
#pragma unroll
        for (int n = 0; n < NK; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[n][e]);
        const float mn = fmaxf(m, half_max(mx) * a.scale2);
        const float mu = mn == -__builtin_inff() ? 0.0f : mn;  // a row that has seen nothing yet
        if (__ballot(mn > m) != 0) {
            const float alpha = exp2_hw(m - mu);
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[dt][e] *= alpha;
        }
        m = mn;
#pragma unroll
        for (int n = 0; n < NK; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[n][e] = exp2_hw(__builtin_fmaf(s[n][e], a.scale2, -mu));
                l += s[n][e];
            }
#pragma unroll
        for (int c = 0; c < 2 * NK; ++c) {
            const Frag<T> p = acc_frag(s[c >> 1], c & 1, T{});
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) mma(o[dt], TL::col_frag(sv, kw0 + 16 * c, dt, lane), p);
        }
    }
    l = half_sum(l);

    if constexpr (WN > 1) {                                     // the waves of a row join their states
        float *js = reinterpret_cast<float *>(smem);
        constexpr int WS = 32 * (DP + 2);
        __syncthreads();
        float *mine = js + (wm * WN + wn) * WS;
        if (h == 0) {
            mine[32 * DP + c32] = m;
            mine[32 * DP + 32 + c32] = l;
        }
        __syncthreads();
        float mt = -__builtin_inff();
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < WN; ++i) mt = fmaxf(mt, js[(wm * WN + i) * WS + 32 * DP + c32]);
        const float mu = mt == -__builtin_inff() ? 0.0f : mt;
#pragma unroll
        for (int i = 0; i < WN; ++i) {
            const float *o1 = js + (wm * WN + i) * WS + 32 * DP + c32;
            l += o1[32] * exp2_hw(o1[0] - mu);
        }
        const float f = exp2_hw(m - mu);
        m = mt;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) mine[(32 * dt + 8 * (e >> 2) + 4 * h + (e & 3)) * 32 + c32] = o[dt][e] * f;
        __syncthreads();
        if (wn) return;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                float x = 0.0f;
#pragma unroll
                for (int i = 0; i < WN; ++i) x += js[(wm * WN + i) * WS + (32 * dt + 8 * (e >> 2) + 4 * h + (e & 3)) * 32 + c32];
                o[dt][e] = x;
            }
    }
    if (!row_ok) return;
    if (STATE || a.splits > 1) {
        const size_t at = (size_t)split * a.Z * a.Lq * (a.KVH * a.G) + row;
        if (h == 0) {
            a.pm[at] = m * LN2;
            a.pl[at] = l;
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const int d = 32 * dt + 8 * b + 4 * h;
                if (d < a.D) store4(a.po + at * a.D + d, o[dt][4 * b], o[dt][4 * b + 1], o[dt][4 * b + 2], o[dt][4 * b + 3]);
            }
    } else {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;          // a row that sees nothing: zeros (NaN stays NaN)
        if (h == 0 && a.lse) a.lse[((size_t)z * a.KVH + kvh) * a.R + rho] = l == 0.0f ? -__builtin_inff() : (m + __log2f(l)) * LN2;
        T *op = static_cast<T *>(a.out) + row * a.D;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const int d = 32 * dt + 8 * b + 4 * h;
                if (d < a.D)
                    store4(op + d, o[dt][4 * b] * inv, o[dt][4 * b + 1] * inv, o[dt][4 * b + 2] * inv, o[dt][4 * b + 3] * inv);
            }
    }
}

// ---------------------------------------------------------------------
// the states of the splits of a row, joined: to a state (out null) or to the row itself.  One wave per row.
// ---------------------------------------------------------------------
struct JoinArgs {
    const float *po, *pm, *pl;
    int splits, D, KVH, G, Lq;
    size_t rows;
    float *so, *sm, *sl;
    void *out;
    float *lse;
};

template <class T>
__global__ void __launch_bounds__(256)
nsd_attn_join_kernel(JoinArgs a)
{
    const int lane = threadIdx.x & 63;
    const size_t row = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= a.rows) return;
    float m = -__builtin_inff();
    for (int s = lane; s < a.splits; s += 64) m = fmaxf(m, a.pm[s * a.rows + row]);
    m = wave_max_f(m);
    const float mu = m == -__builtin_inff() ? 0.0f : m;
    float l = 0.0f;
    for (int s = lane; s < a.splits; s += 64) l += a.pl[s * a.rows + row] * exp2_hw((a.pm[s * a.rows + row] - mu) * LOG2E);
    l = wave_sum_f(l);
    const float inv = a.out ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f;
    for (int d = 2 * lane; d < a.D; d += 128) {
        float x = 0.0f, y = 0.0f;
        for (int s = 0; s < a.splits; ++s) {
            const float f = exp2_hw((a.pm[s * a.rows + row] - mu) * LOG2E);
            const float2 p = *reinterpret_cast<const float2 *>(a.po + (s * a.rows + row) * a.D + d);
            x = __builtin_fmaf(p.x, f, x);
            y = __builtin_fmaf(p.y, f, y);
        }
        x *= inv;
        y *= inv;
        if (a.out) {
            T *o = static_cast<T *>(a.out) + row * a.D + d;
            o[0] = from_f<T>(x);
            o[1] = from_f<T>(y);
        } else {
            *reinterpret_cast<float2 *>(a.so + row * a.D + d) = make_float2(x, y);
        }
    }
    if (lane == 0) {
        if (a.sm) {
            a.sm[row] = m;
            a.sl[row] = l;
        }
        if (a.lse) {
            const int H = a.KVH * a.G, head = (int)(row % H);
            const size_t tok = row / H, z = tok / a.Lq, i = tok % a.Lq;
            a.lse[(z * a.KVH + head / a.G) * ((size_t)a.Lq * a.G) + i * a.G + head % a.G] =
                l == 0.0f ? -__builtin_inff() : m + __log2f(l) * LN2;
        }
    }
}

// ---------------------------------------------------------------------
// backward, first part: dQ = scale dS K with dS = P (dP - delta), dP = dO V^T, delta = rowsum(dO O), which it leaves for
// the second part.  Layout of the forward: a wave owns 32 rows, S^T and dP^T are computed from the same tiles.
// ---------------------------------------------------------------------
template <class T, int DP, int BN>
__global__ void __launch_bounds__(256)
nsd_attn_bwd_q_kernel(SeqArgs a)
{
    constexpr int BM = 128, NK = BN / 32, DT = DP / 32, KC = DP / 16;
    using TL = Tile<T, DP>;
    constexpr int TB = BN * TL::RB;
    __shared__ __align__(16) char smem[4 * TB];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, c32 = lane & 31;
    const int rtiles = (a.R + BM - 1) / BM;
    int bid = blockIdx.x;
    const int rt = rtiles - 1 - bid % rtiles;
    bid /= rtiles;
    const int kvh = bid % a.KVH, z = bid / a.KVH;
    const uint8_t *mask = a.mask ? a.mask + (size_t)z * a.Lk : nullptr;
    const int r0 = rt * BM, rho = r0 + w * 32 + c32;
    const bool row_ok = rho < a.R;
    const int off = a.Lk - a.Lq;
    const int i_row = div_g(row_ok ? rho : a.R - 1, a.g_magic, a.G);
    const int head = kvh * a.G + ((row_ok ? rho : a.R - 1) - i_row * a.G);
    const int last = a.causal ? i_row + off : a.Lk;
    int kend = a.Lk;
    if (a.causal) kend = min(kend, div_g(min(r0 + BM, a.R) - 1, a.g_magic, a.G) + off + 1);
    const int t_end = kend > 0 ? (kend + BN - 1) / BN : 0;
    const T *kb = static_cast<const T *>(a.k) + z * a.k_sz + kvh * a.k_sh;
    const T *vb = static_cast<const T *>(a.v) + z * a.v_sz + kvh * a.v_sh;
    const size_t row = ((size_t)z * a.Lq + i_row) * (a.KVH * a.G) + head;
    const size_t prow = ((size_t)z * a.KVH + kvh) * a.R + rho;

    Frag<T> qf[KC], gf[KC];
    float delta = 0.0f;
    {
        const T *qp = static_cast<const T *>(a.q) + z * a.q_sz + i_row * a.q_st + head * a.q_sh;
        const T *gp = static_cast<const T *>(a.dout) + row * a.D, *op = static_cast<const T *>(a.out) + row * a.D;
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) {
            qf[kc] = mem_frag(qp, 16 * kc + 8 * h, a.D, row_ok);
            gf[kc] = mem_frag(gp, 16 * kc + 8 * h, a.D, row_ok);
            delta = frag_dot(gf[kc], mem_frag(op, 16 * kc + 8 * h, a.D, row_ok), delta);
        }
        delta = half_sum(delta);
    }
    if (h == 0 && row_ok) a.delta[prow] = delta;
    const float lse2 = row_ok ? a.lse[prow] * LOG2E : 0.0f;
    f32x16 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[dt][e] = 0.0f;

    Stage<T, DP, BN> ks, vs;
    uint64_t word = 0, next = 0;
    auto fetch = [&](int tile) {
        const int j0 = tile * BN;
        next = key_word(a, mask, j0, a.Lk);
        auto ok = [&](int r) { return (bool)(next >> (r & 63) & 1); };
        ks.load(kb + (int64_t)j0 * a.k_st, a.k_st, a.D, ok);
        vs.load(vb + (int64_t)j0 * a.v_st, a.v_st, a.D, ok);
    };
    if (t_end > 0) fetch(0);
    for (int t = 0, buf = 0; t < t_end; ++t, buf ^= 1) {
        char *sk = smem + buf * 2 * TB, *sv = sk + TB;
        ks.put(sk);
        vs.put(sv);
        word = next;
        if (t + 1 < t_end) fetch(t + 1);
        __syncthreads();
        const int n_vis = last + 1 - t * BN;
        const uint64_t vis = n_vis <= 0 ? 0 : n_vis < 64 ? word & ((1ull << n_vis) - 1) : word;
#pragma unroll
        for (int n = 0; n < NK; ++n) {
            f32x16 s, dp;
#pragma unroll
            for (int e = 0; e < 16; ++e) { s[e] = 0.0f; dp[e] = -delta; }
#pragma unroll
            for (int kc = 0; kc < KC; ++kc) {
                mma(s, TL::row_frag(sk, 32 * n + c32, kc, h), qf[kc]);
                mma(dp, TL::row_frag(sv, 32 * n + c32, kc, h), gf[kc]);
            }
            const uint32_t bits = (uint32_t)(vis >> (32 * n)) >> (4 * h);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float p = exp2_hw(__builtin_fmaf(s[e], a.scale2, -lse2));
                s[e] = bits >> (8 * (e >> 2) + (e & 3)) & 1 ? p * dp[e] : 0.0f;
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const Frag<T> p = acc_frag(s, c, T{});
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) mma(o[dt], TL::col_frag(sk, 32 * n + 16 * c, dt, lane), p);
            }
        }
    }
    if (!row_ok) return;
    T *op = static_cast<T *>(a.dq) + row * a.D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int d = 32 * dt + 8 * b + 4 * h;
            if (d < a.D)
                store4(op + d, o[dt][4 * b] * a.scale, o[dt][4 * b + 1] * a.scale, o[dt][4 * b + 2] * a.scale,
                       o[dt][4 * b + 3] * a.scale);
        }
}

// ---------------------------------------------------------------------
// backward, second part: dV = P^T dO, dK = scale dS^T Q.  A wave owns 32 keys, whose K and V stay in its registers, and
// the workgroup's four walk over the rows of all G heads (their gradients of a shared head add up in the accumulators):
// S = Q K^T and dP = dO V^T with a lane per key, so that P and dS lie as the B operands of dV^T = dO^T P and
// dK^T = Q^T dS.
// ---------------------------------------------------------------------
template <class T, int DP, int BM>
__global__ void __launch_bounds__(256)
nsd_attn_bwd_kv_kernel(SeqArgs a)
{
    constexpr int BN = 128, NM = BM / 32, DT = DP / 32, KC = DP / 16;
    using TL = Tile<T, DP>;
    constexpr int TB = BM * TL::RB;
    __shared__ __align__(16) char smem[4 * TB];
    __shared__ __align__(16) float stat[2][2][BM];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, c32 = lane & 31;
    const int ktiles = (a.Lk + BN - 1) / BN;
    int bid = blockIdx.x;
    const int kt = bid % ktiles;                                // the first keys are seen by most rows
    bid /= ktiles;
    const int kvh = bid % a.KVH, z = bid / a.KVH;
    const int j = kt * BN + w * 32 + c32;
    bool key_ok = j < a.Lk;
    if (key_ok && a.mask) key_ok = a.mask[(size_t)z * a.Lk + j] != 0;
    const int off = a.Lk - a.Lq;
    const T *kp = static_cast<const T *>(a.k) + z * a.k_sz + kvh * a.k_sh + (int64_t)j * a.k_st;
    const T *vp = static_cast<const T *>(a.v) + z * a.v_sz + kvh * a.v_sh + (int64_t)j * a.v_st;
    Frag<T> kf[KC], vf[KC];
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) {
        kf[kc] = mem_frag(kp, 16 * kc + 8 * h, a.D, key_ok);
        vf[kc] = mem_frag(vp, 16 * kc + 8 * h, a.D, key_ok);
    }
    // rows from first on see this lane's key
    const int64_t lo = a.causal ? (int64_t)(j - off) * a.G : 0;
    const int first = !key_ok ? 0x7fffffff : lo > 0 ? (int)min(lo, (int64_t)a.R) : 0;
    const int64_t lo0 = a.causal ? (int64_t)(kt * BN - off) * a.G : 0;
    const int t_end = (a.R + BM - 1) / BM;
    int t = lo0 > 0 ? (int)min(lo0 / BM, (int64_t)t_end) : 0;

    f32x16 dk[DT], dv[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) { dk[dt][e] = 0.0f; dv[dt][e] = 0.0f; }

    constexpr int PR = TL::PR, U = BM * PR / 256, EP = 16 / (int)sizeof(T);
    uint4 qx[U], gx[U];
    float st_l = 0.0f, st_d = 0.0f;
    const size_t pbase = ((size_t)z * a.KVH + kvh) * a.R;
    auto fetch = [&](int tile) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = (int)threadIdx.x + 256 * u, r = tile * BM + i / PR, p = i % PR;
            qx[u] = gx[u] = make_uint4(0, 0, 0, 0);
            if (r < a.R && p * EP < a.D) {
                const int tok = div_g(r, a.g_magic, a.G), hd = kvh * a.G + r - tok * a.G;
                qx[u] = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.q) + z * a.q_sz + tok * a.q_st + hd * a.q_sh + p * EP);
                gx[u] = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.dout) +
                                                         (((size_t)z * a.Lq + tok) * (a.KVH * a.G) + hd) * a.D + p * EP);
            }
        }
        if (threadIdx.x < BM) {
            const int r = tile * BM + (int)threadIdx.x;
            st_l = r < a.R ? a.lse[pbase + r] * LOG2E : __builtin_inff();       // no row: probability 0
            st_d = r < a.R ? a.delta[pbase + r] : 0.0f;
        }
    };
    if (t < t_end) fetch(t);
    for (int buf = 0; t < t_end; ++t, buf ^= 1) {
        char *sq = smem + buf * 2 * TB, *sg = sq + TB;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = (int)threadIdx.x + 256 * u;
            *reinterpret_cast<uint4 *>(sq + TL::at(i / PR, i % PR)) = qx[u];
            *reinterpret_cast<uint4 *>(sg + TL::at(i / PR, i % PR)) = gx[u];
        }
        if (threadIdx.x < BM) {
            stat[buf][0][threadIdx.x] = st_l;
            stat[buf][1][threadIdx.x] = st_d;
        }
        if (t + 1 < t_end) fetch(t + 1);
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NM; ++n) {
            f32x16 s, dp;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const float4 x = *reinterpret_cast<const float4 *>(&stat[buf][1][32 * n + 8 * b + 4 * h]);
                dp[4 * b] = -x.x; dp[4 * b + 1] = -x.y; dp[4 * b + 2] = -x.z; dp[4 * b + 3] = -x.w;
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = 0.0f;
#pragma unroll
            for (int kc = 0; kc < KC; ++kc) {
                mma(s, TL::row_frag(sq, 32 * n + c32, kc, h), kf[kc]);
                mma(dp, TL::row_frag(sg, 32 * n + c32, kc, h), vf[kc]);
            }
            const int thr = first - (t * BM + 32 * n + 4 * h);
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const float4 x = *reinterpret_cast<const float4 *>(&stat[buf][0][32 * n + 8 * b + 4 * h]);
                const float ls[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float p = exp2_hw(__builtin_fmaf(s[4 * b + e], a.scale2, -ls[e]));
                    s[4 * b + e] = 8 * b + e >= thr ? p : 0.0f;
                    dp[4 * b + e] = 8 * b + e >= thr ? p * dp[4 * b + e] : 0.0f;
                }
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const Frag<T> p = acc_frag(s, c, T{}), ds = acc_frag(dp, c, T{});
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    mma(dv[dt], TL::col_frag(sg, 32 * n + 16 * c, dt, lane), p);
                    mma(dk[dt], TL::col_frag(sq, 32 * n + 16 * c, dt, lane), ds);
                }
            }
        }
    }
    if (j >= a.Lk) return;
    const size_t at = (((size_t)z * a.Lk + j) * a.KVH + kvh) * a.D;
    T *pk = static_cast<T *>(a.dk) + at, *pv = static_cast<T *>(a.dv) + at;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int d = 32 * dt + 8 * b + 4 * h;
            if (d >= a.D) continue;
            float x[4], y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {                       // a masked key has no part in anything
                x[e] = key_ok ? dk[dt][4 * b + e] * a.scale : 0.0f;
                y[e] = key_ok ? dv[dt][4 * b + e] : 0.0f;
            }
            store4(pk + d, x[0], x[1], x[2], x[3]);
            store4(pv + d, y[0], y[1], y[2], y[3]);
        }
}

// ---------------------------------------------------------------------
// launchers
// ---------------------------------------------------------------------
constexpr int CUS = 256;

struct FwdPlan { int wm, bn, rtiles, splits, split_tiles; };

int dp_of(int D) { return D <= 64 ? 64 : 128; }

// Row tiles of 128 (four waves along the rows) unless there are at most 64 or 32 rows: the waves then share the keys of
// a tile.  The keys are split over several workgroups while there are fewer workgroups than CUs.
FwdPlan fwd_plan(int Z, int KVH, int R, int Lk, int D, int dtype)
{
    FwdPlan p;
    p.wm = R <= 32 ? 1 : R <= 64 ? 2 : 4;
    const int kw = dtype == 0 ? 32 : p.wm == 1 ? 32 : 64;
    p.bn = kw * (4 / p.wm);
    p.rtiles = (R + 32 * p.wm - 1) / (32 * p.wm);
    const int64_t wgs = (int64_t)p.rtiles * KVH * Z;
    const int tiles = (Lk + p.bn - 1) / p.bn;
    p.splits = 1;
    if (wgs < CUS && tiles > 1) {
        int64_t s = (2 * CUS + wgs - 1) / wgs;
        s = s < tiles ? s : tiles;
        p.split_tiles = (int)((tiles + s - 1) / s);
        p.splits = (tiles + p.split_tiles - 1) / p.split_tiles;
    } else {
        p.split_tiles = tiles > 0 ? tiles : 1;
    }
    return p;
}

template <class T, int DP, bool STATE>
void launch_fwd(const SeqArgs &a, const FwdPlan &p, hipStream_t s)
{
    constexpr bool F = sizeof(T) == 4;
    const dim3 grid((unsigned)((int64_t)p.rtiles * a.KVH * a.Z * p.splits)), block(256);
    if (p.wm == 4) hipLaunchKernelGGL((nsd_attn_fwd_kernel<T, DP, 4, F ? 32 : 64, 2, STATE>), grid, block, 0, s, a);
    else if (p.wm == 2) hipLaunchKernelGGL((nsd_attn_fwd_kernel<T, DP, 2, F ? 32 : 64, F && DP == 128 ? 2 : 1, STATE>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((nsd_attn_fwd_kernel<T, DP, 1, 32, F && DP == 128 ? 1 : 2, STATE>), grid, block, 0, s, a);
}

int run_join(const JoinArgs &j, int dtype, hipStream_t s)
{
    const dim3 grid((unsigned)((j.rows + 3) / 4)), block(256);
    if (dtype == 0) hipLaunchKernelGGL(nsd_attn_join_kernel<float>, grid, block, 0, s, j);
    else hipLaunchKernelGGL(nsd_attn_join_kernel<BF16>, grid, block, 0, s, j);
    return (int)hipGetLastError();
}

template <bool STATE>
int run_fwd(const SeqArgs &a, const FwdPlan &p, int dtype, hipStream_t s)
{
    if (dtype == 0) {
        if (dp_of(a.D) == 64) launch_fwd<float, 64, STATE>(a, p, s);
        else launch_fwd<float, 128, STATE>(a, p, s);
    } else {
        if (dp_of(a.D) == 64) launch_fwd<BF16, 64, STATE>(a, p, s);
        else launch_fwd<BF16, 128, STATE>(a, p, s);
    }
    return (int)hipGetLastError();
}

template <class T, int DP>
void launch_bwd(const SeqArgs &a, hipStream_t s)
{
    constexpr int BN = sizeof(T) == 4 && DP == 128 ? 32 : 64;
    const dim3 block(256);
    if (a.R > 0)
        hipLaunchKernelGGL((nsd_attn_bwd_q_kernel<T, DP, BN>), dim3((unsigned)((int64_t)((a.R + 127) / 128) * a.KVH * a.Z)), block, 0, s, a);
    if (a.Lk > 0)
        hipLaunchKernelGGL((nsd_attn_bwd_kv_kernel<T, DP, 32>), dim3((unsigned)((int64_t)((a.Lk + 127) / 128) * a.KVH * a.Z)), block, 0, s, a);
}

bool al16(const void *p) { return ((uintptr_t)p & 15u) == 0; }

// the shape fields that the entry points share, checked; strides in pieces of 16 bytes
int seq_args(const NsdSeqAttn *p, const void *q, const void *k, const void *v, SeqArgs &a)
{
    if (!p) return NSD_E_NULL;
    if (p->batch < 0 || p->len_q < 0 || p->len_k < 0 || p->heads < 1 || p->kv_heads < 1 || p->heads % p->kv_heads ||
        p->hd < 8 || p->hd > 128 || p->hd % 8 || (p->dtype != 0 && p->dtype != 1))
        return NSD_E_SIZE;
    if (!(p->scale > 0.0f) || p->scale > 3.0e38f) return NSD_E_SIZE;
    const int64_t G = p->heads / p->kv_heads, R = (int64_t)p->len_q * G;
    // rho / G by multiplication is exact while R * G < 2^32; tile and grid indices are 32-bit
    if (R > (1ll << 30) || R * G >= (1ll << 32) || p->len_k > (1 << 30)) return NSD_E_SIZE;
    const int64_t zk = (int64_t)p->batch * p->kv_heads;
    if (zk * ((R + 31) / 32) > (1ll << 30) || zk * (((int64_t)p->len_k + 31) / 32) > (1ll << 30)) return NSD_E_SIZE;
    if (p->batch == 0) return NSD_OK;
    const int ep = p->dtype ? 8 : 4;
    for (int i = 0; i < 3; ++i)
        if (p->q_stride[i] % ep || p->k_stride[i] % ep || p->v_stride[i] % ep) return NSD_E_ALIGN;
    if (!al16(q) || !al16(k) || !al16(v)) return NSD_E_ALIGN;
    if ((R > 0 && !q) || (p->len_k > 0 && (!k || !v))) return NSD_E_NULL;
    a = SeqArgs{};
    a.q = q; a.k = k; a.v = v;
    a.q_sz = p->q_stride[0]; a.q_st = p->q_stride[1]; a.q_sh = p->q_stride[2];
    a.k_sz = p->k_stride[0]; a.k_st = p->k_stride[1]; a.k_sh = p->k_stride[2];
    a.v_sz = p->v_stride[0]; a.v_st = p->v_stride[1]; a.v_sh = p->v_stride[2];
    a.mask = p->key_mask; a.lens = p->key_len;
    a.Z = p->batch; a.KVH = p->kv_heads; a.G = (int)G; a.Lq = p->len_q; a.Lk = p->len_k; a.D = p->hd; a.R = (int)R;
    a.causal = p->causal ? 1 : 0;
    a.g_magic = (uint32_t)(((1ull << 32) + G - 1) / G);
    a.scale = p->scale;
    a.scale2 = p->scale * LOG2E;
    a.splits = 1;
    return NSD_OK;
}

size_t state_bytes(const SeqArgs &a) { return (size_t)a.Z * a.Lq * a.KVH * a.G * ((size_t)a.D + 2) * 4; }

} // namespace

extern "C" int64_t nsd_attn_fwd_workspace(const NsdSeqAttn *p)
{
    if (!p || p->kv_heads < 1 || p->heads < 1 || p->hd < 1 || p->batch < 1 || p->len_q < 1) return 0;
    const int G = p->heads / p->kv_heads;
    const FwdPlan f = fwd_plan(p->batch, p->kv_heads, p->len_q * G, p->len_k, p->hd, p->dtype);
    return f.splits > 1 ? (int64_t)f.splits * p->batch * p->len_q * p->heads * (p->hd + 2) * 4 : 0;
}

extern "C" int nsd_attn_fwd(const void *q, const void *k, const void *v, const NsdSeqAttn *p, void *out, float *lse,
                            void *ws, int64_t ws_bytes, void *stream)
{
    SeqArgs a;
    if (const int rc = seq_args(p, q, k, v, a)) return rc;
    if (p->batch == 0 || p->len_q == 0) return NSD_OK;
    if (!out) return NSD_E_NULL;
    if (!al16(out) || !al16(ws)) return NSD_E_ALIGN;
    const FwdPlan f = fwd_plan(a.Z, a.KVH, a.R, a.Lk, a.D, p->dtype);
    a.splits = f.splits;
    a.split_tiles = f.split_tiles;
    a.out = out;
    a.lse = lse;
    if (f.splits > 1) {
        if (!ws) return NSD_E_NULL;
        if (ws_bytes < (int64_t)(f.splits * state_bytes(a))) return NSD_E_SIZE;
        const size_t rows = (size_t)a.Z * a.Lq * a.KVH * a.G;
        a.po = (float *)ws;
        a.pm = a.po + f.splits * rows * a.D;
        a.pl = a.pm + f.splits * rows;
    }
    if (const int rc = run_fwd<false>(a, f, p->dtype, (hipStream_t)stream)) return rc;
    if (f.splits == 1) return NSD_OK;
    JoinArgs j{a.po, a.pm, a.pl, f.splits, a.D, a.KVH, a.G, a.Lq, (size_t)a.Z * a.Lq * a.KVH * a.G, nullptr, nullptr, nullptr, out, lse};
    return run_join(j, p->dtype, (hipStream_t)stream);
}

extern "C" int64_t nsd_attn_bwd_workspace(const NsdSeqAttn *p)
{
    if (!p || p->batch < 1 || p->len_q < 1 || p->heads < 1) return 0;
    return (int64_t)p->batch * p->len_q * p->heads * 4;
}

extern "C" int nsd_attn_bwd(const void *q, const void *k, const void *v, const void *out, const float *lse, const void *dout,
                            const NsdSeqAttn *p, void *dq, void *dk, void *dv, void *ws, int64_t ws_bytes, void *stream)
{
    SeqArgs a;
    if (const int rc = seq_args(p, q, k, v, a)) return rc;
    if (p->key_len) return NSD_E_SIZE;                          // ragged keys are a form of the prefix state only
    if (p->batch == 0) return NSD_OK;
    if (a.R > 0 && (!out || !lse || !dout || !dq || !ws)) return NSD_E_NULL;
    if (a.Lk > 0 && (!dk || !dv)) return NSD_E_NULL;
    if (!al16(out) || !al16(dout) || !al16(dq) || !al16(dk) || !al16(dv) || !al16(ws)) return NSD_E_ALIGN;
    if (ws_bytes < (int64_t)a.Z * a.KVH * a.R * 4) return NSD_E_SIZE;
    a.out = const_cast<void *>(out);
    a.lse = const_cast<float *>(lse);
    a.dout = dout;
    a.delta = (float *)ws;
    a.dq = dq; a.dk = dk; a.dv = dv;
    if (p->dtype == 0) {
        if (dp_of(a.D) == 64) launch_bwd<float, 64>(a, (hipStream_t)stream);
        else launch_bwd<float, 128>(a, (hipStream_t)stream);
    } else {
        if (dp_of(a.D) == 64) launch_bwd<BF16, 64>(a, (hipStream_t)stream);
        else launch_bwd<BF16, 128>(a, (hipStream_t)stream);
    }
    return (int)hipGetLastError();
}

extern "C" int64_t nsd_attn_prefix_workspace(const NsdSeqAttn *p)
{
    return nsd_attn_fwd_workspace(p);
}

extern "C" int nsd_attn_prefix(const void *q, const void *k, const void *v, const NsdSeqAttn *p, int32_t has_state,
                               float *part_o, float *part_m, float *part_l, void *ws, int64_t ws_bytes, void *stream)
{
    SeqArgs a;
    if (const int rc = seq_args(p, q, k, v, a)) return rc;
    if (p->causal || p->key_mask) return NSD_E_SIZE;            // every hypothesis sees the whole prefix
    if (p->batch == 0 || p->len_q == 0) return NSD_OK;
    if (!part_o || !part_m || !part_l) return NSD_E_NULL;
    if (!al16(part_o) || !al16(ws)) return NSD_E_ALIGN;
    const FwdPlan f = fwd_plan(a.Z, a.KVH, a.R, a.Lk, a.D, p->dtype);
    const size_t rows = (size_t)a.Z * a.Lq * a.KVH * a.G;
    a.splits = f.splits;
    a.split_tiles = f.split_tiles;
    if (has_state) { a.in_o = part_o; a.in_m = part_m; a.in_l = part_l; }
    a.po = part_o; a.pm = part_m; a.pl = part_l;
    if (f.splits > 1) {
        if (!ws) return NSD_E_NULL;
        if (ws_bytes < (int64_t)(f.splits * state_bytes(a))) return NSD_E_SIZE;
        a.po = (float *)ws;
        a.pm = a.po + f.splits * rows * a.D;
        a.pl = a.pm + f.splits * rows;
    }
    if (const int rc = run_fwd<true>(a, f, p->dtype, (hipStream_t)stream)) return rc;
    if (f.splits == 1) return NSD_OK;
    JoinArgs j{a.po, a.pm, a.pl, f.splits, a.D, a.KVH, a.G, a.Lq, rows, part_o, part_m, part_l, nullptr, nullptr};
    return run_join(j, p->dtype, (hipStream_t)stream);
}
