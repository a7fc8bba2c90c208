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
// gradients are rounded to bf16 only where they enter a bf16 product.  That takes the error of a result against 64 bits from
// 1.65e-3 of its size (its own rounding) to 1.9e-3, and of a gradient to 2.4e-3.  A second product with what the rounding
// left (rest_frag) takes it back for a third to a half more matrix instructions: done in the backward pass where a launch
// waits on latencies and has them free (FINE), so the last bits of a sequence's gradients depend on how many sequences share
// its batch.
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
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

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

// what that rounding left of them, as an operand of its own: with both, a product sees 16 bits of the accumulator
NSD_D Frag<BF16> rest_frag(const f32x16 &s, int c, const Frag<BF16> &hi)
{
    f32x16 r = s;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[8 * c + j] = s[8 * c + j] - (float)hi.v[j];
    return acc_frag(r, c, BF16{});
}
NSD_D Frag<float> rest_frag(const f32x16 &, int, const Frag<float> &f) { return f; }

// Order for the compiler's scheduler: AHEAD operand reads from LDS before the first of MFMAS matrix instructions, then READS
// more after each.  Left to itself it reads every operand into the same registers right before its use, and each matrix
// instruction waits out an LDS latency: dQ of one sequence of 8192 took 645 us, 592 in this order.  (The forward pass is the
// same in either; dK and dV have no registers left for it.)
template <int MFMAS, int READS, int AHEAD> NSD_D void feed()
{
    __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
    for (int i = 0; i < MFMAS; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if (AHEAD + READS * i < MFMAS * READS) __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    }
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

// A tile of rows in LDS, DP elements each, in 16-byte pieces, as chunks of 16 rows x 4 pieces (1 KiB, what a wave fetches
// with one instruction, 64 bytes of a row by four adjacent lanes).  Piece p of row r lies at place p ^ g(r) of its row's
// four: sixteen lanes that read one piece of sixteen rows (the operand reads along a row) touch all 64 banks once, and so
// do the 32 lanes that read 32 bytes of eight rows (the transposing reads).  Whole chunks are a constant apart, so an
// operand's many reads are few address registers and immediate offsets (with a swizzle across the whole row every one
// had an address of its own: 20 registers, which the kernels' two waves per SIMD do not have).
template <class T, int DP> struct Tile {
    static constexpr int RB = DP * (int)sizeof(T);              // bytes of a row
    static constexpr int PR = RB / 16;                          // pieces of a row
    static constexpr int CG = PR / 4;                           // chunks of 16 rows
    static constexpr bool B16 = sizeof(T) == 2;
    NSD_D static int g(int r) { return (r >> 1 & 3) ^ (r >> 3 & 1); }

    // elements 16 kc + 8 h .. + 7 of row row0 + c32 (row0 a multiple of 32; lane = 32 h + c32)
    NSD_D static Frag<T> row_frag(const char *s, int row0, int kc, int lane)
    {
        Frag<T> f;
        const int c32 = lane & 31, h = lane >> 5, r = c32 & 15;
        const char *p = s + ((row0 >> 4) + (c32 >> 4)) * (CG * 1024) + r * 64;
        if constexpr (B16) {
            const int x = ((h ^ g(r)) << 4) ^ ((kc & 1) << 5);
            f.v = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4 *>(p + x + (kc >> 1) * 1024));
        } else {
            const int x = (2 * h ^ g(r)) << 4;
            const float4 u = *reinterpret_cast<const float4 *>(p + x + kc * 1024);
            const float4 v = *reinterpret_cast<const float4 *>(p + (x ^ 16) + kc * 1024);
            f.v[0] = u.x; f.v[1] = u.y; f.v[2] = u.z; f.v[3] = u.w;
            f.v[4] = v.x; f.v[5] = v.y; f.v[6] = v.z; f.v[7] = v.w;
        }
        return f;
    }
    // column 32 dt + (lane & 31) of rows r0 + 4 h + 0..3 and r0 + 8 + 4 h + 0..3 (r0 a multiple of 16)
    NSD_D static Frag<T> col_frag(const char *s, int r0, int dt, int lane)
    {
        Frag<T> f;
        const int h = lane >> 5;
        const char *p = s + (r0 >> 4) * (CG * 1024);
        if constexpr (B16) {
            // sixteen lanes hand in 32 bytes of four rows and get a column of sixteen each
            const int r = 4 * h + (lane >> 2 & 3), piece = 2 * (lane >> 4 & 1) + (lane >> 1 & 1);
            const int x = ((piece ^ g(r)) << 4) + 8 * (lane & 1);
            typedef __attribute__((address_space(3))) s16x4 lds4;
            const s16x4 u = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)(p + r * 64 + x + dt * 1024));
            const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)(p + r * 64 + (x ^ 16) + 512 + dt * 1024));
            f.v = __builtin_bit_cast(bf16x8, __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            const int piece = lane >> 2 & 3;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int r = 8 * (j >> 2) + 4 * h + (j & 3);
                f.v[j] = *reinterpret_cast<const float *>(p + (2 * dt + (lane >> 4 & 1)) * 1024 + r * 64 + ((piece ^ g(r)) << 4) + 4 * (lane & 3));
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

// What rounding to bf16 took from a value, in 256ths of the last place that bf16 keeps, plus 128: a byte, with which the
// row sums dO . O of the backward pass see 16 bits of O.  (With bf16's 8 alone the error of dQ and dK grows by up to 1.3
// times, most at short rows; the rest in bf16 is twice the traffic.)
NSD_D uint32_t rest4(float a, float b, float c, float d)
{
    const float v[4] = {a, b, c, d};
    uint32_t r = 0;
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
        const f32x2 x = {v[j], v[j + 1]};
        const uint32_t u = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf16x2));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t hi = i ? u & 0xffff0000u : u << 16;
            // 2^15 / 2^exponent, of 2^-111 for what is below it: rest_dot then takes less of the rest than there was, by 2^-120
            // at most
            const float inv = __uint_as_float(max(0x7f000000u + (15u << 23) - max(hi & 0x7f800000u, 16u << 23), 0u));
            r = __builtin_amdgcn_cvt_pk_u8_f32(__builtin_fmaf(v[j + i] - __uint_as_float(hi), inv, 128.0f), j + i, r);
        }
    }
    return r;
}
// sum of g times the rest of o over a lane's eight elements
NSD_D float rest_dot(const Frag<BF16> &g, const Frag<BF16> &o, const uint8_t *rest, float s)
{
    const uint2 c = *reinterpret_cast<const uint2 *>(rest);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float b = (float)((j < 4 ? c.x : c.y) >> (8 * (j & 3)) & 255u) - 128.0f;
        const float f = __uint_as_float(__float_as_uint((float)o.v[j]) & 0x7f800000u);
        s = __builtin_fmaf((float)g.v[j] * f, b * (1.0f / 32768.0f), s);
    }
    return s;
}
NSD_D float rest_dot(const Frag<float> &, const Frag<float> &, const uint8_t *, float s) { return s; }

// A wave's 32 rows from its transposed accumulators (lane = row, registers = elements) to memory, times `mul`.  bf16 rows
// pass through LDS (`s`, the wave's own 32 * (RB + 16) bytes) and leave in 16-byte pieces of whole rows: stored from the
// accumulators they would be 8 bytes here and there, 16 stores that touch 32 rows each.  The stores pass by the caches,
// which the keys need (32 x 768 positions: 212 -> 187 us).  ptr(r) is row r's place or null.
template <class T, int DP, class P>
NSD_D void put_rows(char *s, const f32x16 (&o)[DP / 32], float mul, int D, int lane, P ptr)
{
    const int c32 = lane & 31, h = lane >> 5;
    if constexpr (sizeof(T) == 2) {
        constexpr int PR = DP / 8, SB = DP * 2 + 16;
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
            for (int b = 0; b < 4; ++b)
                store4(reinterpret_cast<T *>(s + c32 * SB) + 32 * dt + 8 * b + 4 * h, o[dt][4 * b] * mul, o[dt][4 * b + 1] * mul,
                       o[dt][4 * b + 2] * mul, o[dt][4 * b + 3] * mul);
        nsd_wave_sync();
#pragma unroll
        for (int i = 0; i < 32 * PR / 64; ++i) {
            const int r = (i * 64 + lane) / PR, p = (i * 64 + lane) % PR;
            T *dst = ptr(r);
            if (dst && p * 8 < D)
                __builtin_nontemporal_store(*reinterpret_cast<const u32x4 *>(s + r * SB + p * 16), reinterpret_cast<u32x4 *>(dst + p * 8));
        }
        nsd_wave_sync();
    } else {
        T *dst = ptr(c32);
        if (!dst) return;
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const int d = 32 * dt + 8 * b + 4 * h;
                if (d < D) store4(dst + d, o[dt][4 * b] * mul, o[dt][4 * b + 1] * mul, o[dt][4 * b + 2] * mul, o[dt][4 * b + 3] * mul);
            }
    }
}
// The rows' rests, a byte an element, the same way (bf16 only).
template <int DP, class P>
NSD_D void put_rest(char *s, const f32x16 (&o)[DP / 32], float mul, int D, int lane, P ptr)
{
    const int c32 = lane & 31, h = lane >> 5;
    constexpr int PR = DP / 8, SB = DP + 16;
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int b = 0; b < 4; ++b)
            *reinterpret_cast<uint32_t *>(s + c32 * SB + 32 * dt + 8 * b + 4 * h) =
                rest4(o[dt][4 * b] * mul, o[dt][4 * b + 1] * mul, o[dt][4 * b + 2] * mul, o[dt][4 * b + 3] * mul);
    nsd_wave_sync();
#pragma unroll
    for (int i = 0; i < 32 * PR / 64; ++i) {
        const int r = (i * 64 + lane) / PR, p = (i * 64 + lane) % PR;
        uint8_t *dst = ptr(r);
        if (dst && p * 8 < D)
            __builtin_nontemporal_store(*reinterpret_cast<const u32x2 *>(s + r * SB + p * 8), reinterpret_cast<u32x2 *>(dst + p * 8));
    }
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
    uint8_t *rest;                         // a byte for each element of out, or null: see rest4
    float *po, *pm, *pl;                   // state [splits][Z * Lq * heads] (sum of weighted values, maximum, sum)
    const float *in_o, *in_m, *in_l;       // a state to continue, or null
    int splits, split_tiles, batch;
    // backward
    const void *dout;                      // [Z, Lq, heads, D]
    float *delta;                          // [Z, KVH, R]
    void *dq, *dk, *dv;                    // contiguous like q, k, v
    float *part, *part_v;                  // splits > 1: fp32 sums of dq, or of dk and dv, [splits] of them
    float scale;
};

NSD_D int div_g(int rho, uint32_t magic, int G) { return G == 1 ? rho : (int)(((uint64_t)(uint32_t)rho * magic) >> 32); }

// Work of a workgroup: which of `tiles` of which of `pairs` (batch, kv head and split of its keys).  Workgroups go to the
// eight XCDs in turn, each with an L2 of its own: where the pairs divide evenly every XCD takes whole pairs, so that the
// tiles of a pair share its L2, `batch` pairs at a time (enough to fill the XCD), and among those the costly tiles first.
NSD_D void work_of(int bid, int tiles, int pairs, int batch, int &pair, int &tile)
{
    const int xcds = pairs % 8 == 0 ? 8 : 1, per = pairs / xcds;
    const int x = bid % xcds, i = bid / xcds;
    const int first = i / (batch * tiles) * batch, n = min(batch, per - first), j = i - first * tiles;
    pair = (first + j % n) * xcds + x;
    tile = j / n;
}

// The keys of a tile that exist and are not masked, as words that every lane has.  A lane asks for its key's mask byte a
// tile before the word is needed, so that no tile waits for it.
template <int NW> struct KeyMask {
    const uint8_t *mask;
    int n_keys;
    uint32_t byte[NW];
    NSD_D void ask(int j0)
    {
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            const int j = j0 + 64 * i + (int)(threadIdx.x & 63);
            byte[i] = j < n_keys ? 1 : 0;
            if (mask && j < n_keys) byte[i] = mask[j];
        }
    }
    // (a tile of 32 keys uses the lower half of its word)
    NSD_D bool words(uint64_t (&w)[NW], uint64_t part) const
    {
        uint64_t any = 0;
#pragma unroll
        for (int i = 0; i < NW; ++i) any |= w[i] = __ballot(byte[i] != 0) & part;
        return any != 0;
    }
};

// A tile of ROWS rows goes from memory straight to LDS (global_load_lds), 16 bytes a lane and instruction: a wave fills
// 1 KiB in lane order, so the piece that a lane fetches is the one that the swizzle puts at its place.  Rows that are
// not there, and pieces past a row's D elements, come from a page of zeros: no query may see what lies there, not even
// as 0 * NaN.  The load is written out because the compiler, which cannot tell the two halves of the double buffer
// apart, would wait for it before the next transposing read of the other half; tile_barrier() is the wait.
__device__ const uint4 zero_page[1] = {};

NSD_D void to_lds(uint64_t g, uint32_t lds)
{
    uint32_t m0;                                                // left as it was: the compiler may keep a value of its own there
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(m0) : "v"(g), "s"(lds) : "memory");
}
// every wave's loads have arrived, and every wave is done with what they will overwrite next
NSD_D void tile_barrier()
{
    asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
    __syncthreads();
}
NSD_D uint32_t lds_at(const char *p)
{
    typedef __attribute__((address_space(3))) const char lds_char;
    return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_char *)p);
}

// This lane's part of a tile of ROWS rows: the wave fetches chunks w + 4 u, of which the lane fetches one piece.
template <class T, int DP, int ROWS> struct Stage {
    static constexpr int CG = Tile<T, DP>::CG, U = ROWS / 16 * CG / 4, EP = 16 / (int)sizeof(T);
    int w, row, elem;                                           // row in a chunk, element in a chunk's rows
    NSD_D Stage()
    {
        const int lane = threadIdx.x & 63;
        w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        row = lane >> 2;
        elem = ((lane & 3) ^ Tile<T, DP>::g(row)) * EP;
    }
    NSD_D int chunk_row(int u) const { return (w + 4 * u) / CG * 16; }
    NSD_D int chunk_elem(int u) const { return (w + 4 * u) % CG * 4 * EP; }
    NSD_D uint32_t place(uint32_t tile, int u) const { return tile + (w + 4 * u) * 1024; }
    // rows of `base`, `stride` elements apart; row r of the tile is there if bit r of `words` is set
    template <int NW> NSD_D void load(const T *base, int64_t stride, int D, const uint64_t (&words)[NW], const char *tile) const
    {
        const uint64_t p = (uint64_t)(base + row * stride + elem), zero = (uint64_t)zero_page;
        const uint32_t dst = lds_at(tile);
        bool whole = D == DP;
#pragma unroll
        for (int i = 0; i < NW; ++i) whole = whole && words[i] == (ROWS < 64 ? (1ull << (ROWS & 63)) - 1 : ~0ull);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            uint64_t q = p + (uint64_t)(chunk_row(u) * stride + chunk_elem(u)) * sizeof(T);
            if (!whole) {
                const int r = chunk_row(u) + row;
                const bool ok = chunk_elem(u) + elem < D && (words[NW > 1 ? r >> 6 : 0] >> (r & 63) & 1);
                q = ok ? q : zero;
            }
            to_lds(q, place(dst, u));
        }
    }
};

// ---------------------------------------------------------------------
// forward.  A workgroup of four waves: WM of them along the rows (32 each), WN = 4 / WM along the keys (KW of a tile's
// BN = KW * WN each; their states meet at the end).  grid.x = row tile, (z, kv head), split.
// ---------------------------------------------------------------------
template <class T, int DP, int WM, int KW, int NBUF, bool STATE>
__global__ void __launch_bounds__(256, sizeof(T) == 2 && 2 * NBUF * KW * (4 / WM) * DP * 2 <= 81920 ? 2 : 1)
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
    int pair, tile;
    work_of(blockIdx.x, rtiles, a.Z * a.KVH * a.splits, a.batch, pair, tile);
    const int rt = rtiles - 1 - tile;                           // later rows of a causal mask see more keys
    const int split = pair % a.splits, kvh = pair / a.splits % a.KVH, z = pair / a.splits / a.KVH;
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
    constexpr uint64_t PART = BN < 64 ? (1ull << (BN & 63)) - 1 : ~0ull;
    KeyMask<NW> keys{mask, n_keys, {}};
    if (t < t_end) keys.ask(t * BN);
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

    // Double buffer: while a tile is worked on, the next one is on its way, and the mask bytes of the one after that.
    uint64_t word[NW], next[NW];
    bool any = false, next_any = false;                         // tiles without a visible key are passed over
    const Stage<T, DP, BN> stage;
    auto fetch = [&](int tile, const char *s) {
        next_any = keys.words(next, PART);
        if (next_any) {
            stage.load(kb + (int64_t)tile * BN * a.k_st, a.k_st, a.D, next, s);
            stage.load(vb + (int64_t)tile * BN * a.v_st, a.v_st, a.D, next, s + TB);
        }
        keys.ask((tile + 1) * BN);
    };
    if (NBUF == 2 && t < t_end) fetch(t, smem);
    for (int buf = 0; t < t_end; ++t, buf ^= NBUF - 1) {
        const char *sk = smem + buf * 2 * TB, *sv = sk + TB;
        if (NBUF == 1) {
            __syncthreads();                                    // everyone has read the last tile
            fetch(t, smem);
        }
        tile_barrier();                                         // the tile is there (and the other buffer free)
        any = next_any;
#pragma unroll
        for (int i = 0; i < NW; ++i) word[i] = next[i];
        if (NBUF == 2 && t + 1 < t_end) fetch(t + 1, smem + (buf ^ 1) * 2 * TB);
        if (!any) continue;

        // scores of this wave's KW keys
        f32x16 s[NK];
#pragma unroll
        for (int n = 0; n < NK; ++n) {
#pragma unroll
            for (int e = 0; e < 16; ++e) s[n][e] = 0.0f;
#pragma unroll
            for (int kc = 0; kc < KC; ++kc) mma(s[n], TL::row_frag(sk, wn * KW + 32 * n, kc, lane), qf[kc]);
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
        // (A reference that follows the maximum only from afar saves most of the rescaling, 437 -> 421 us for one sequence
        // of 8192, but the weight of the leading key is then no longer the 1 that bf16 holds exactly: the error of the
        // result grows from 1.9e-3 to 2.5e-3 of its size.  Not kept.)
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
    if (STATE || a.splits > 1) {
        const size_t at = (size_t)split * a.Z * a.Lq * (a.KVH * a.G) + row;
        if (h == 0 && row_ok) {
            a.pm[at] = m * LN2;
            a.pl[at] = l;
        }
        put_rows<float, DP>(nullptr, o, 1.0f, a.D, lane, [&](int) { return row_ok ? a.po + at * a.D : nullptr; });
    } else {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;          // a row that sees nothing: zeros (NaN stays NaN)
        if (h == 0 && row_ok && a.lse)
            a.lse[((size_t)z * a.KVH + kvh) * a.R + rho] = l == 0.0f ? -__builtin_inff() : (m + __log2f(l)) * LN2;
        if (WN == 1) __syncthreads();                           // everyone is done with the tiles
        char *mine = smem + wm * (WN > 1 ? WN * 32 * (DP + 2) * 4 : 32 * (DP * 2 + 16));    // (what only this wave has read)
        auto place = [&](int r) {                               // of row r of the wave's 32, in elements; -1: no row
            const int x = r0 + wm * 32 + r, i = div_g(x, a.g_magic, a.G);
            return x < a.R ? (int64_t)((((size_t)z * a.Lq + i) * a.KVH + kvh) * a.G + (x - i * a.G)) * a.D : -1;
        };
        put_rows<T, DP>(mine, o, inv, a.D, lane, [&](int r) { const int64_t x = place(r); return x < 0 ? nullptr : static_cast<T *>(a.out) + x; });
        if constexpr (sizeof(T) == 2) {
            if (a.rest) put_rest<DP>(mine, o, inv, a.D, lane, [&](int r) { const int64_t x = place(r); return x < 0 ? nullptr : a.rest + x; });
        }
    }
}

// ---------------------------------------------------------------------
// the states of the splits of a row, joined: to a state (out null) or to the row itself.  32 lanes hold a row's D
// elements, `share` such groups (a power of two) share the splits of a row, so that a workgroup of eight groups has many
// loads on their way where a row has many splits and works on several rows where it has few.
// ---------------------------------------------------------------------
struct JoinArgs {
    const float *po, *pm, *pl;
    int splits, D, KVH, G, Lq, share;
    size_t rows;
    float *so, *sm, *sl;
    void *out;
    uint8_t *rest;
    float *lse;
};

template <class T>
__global__ void __launch_bounds__(256)
nsd_attn_join_kernel(JoinArgs a)
{
    __shared__ __align__(16) float4 sum[8][32];
    const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5, part = grp % a.share;
    const size_t row = (size_t)blockIdx.x * (8 / a.share) + grp / a.share;
    const bool row_ok = row < a.rows;
    float m = -__builtin_inff(), l = 0.0f, mu = 0.0f;
    float4 x = make_float4(0, 0, 0, 0);
    if (row_ok) {
        for (int s = lane; s < a.splits; s += 32) m = fmaxf(m, a.pm[s * a.rows + row]);
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, 32));
        mu = m == -__builtin_inff() ? 0.0f : m;
        for (int s = lane; s < a.splits; s += 32) l += a.pl[s * a.rows + row] * exp2_hw((a.pm[s * a.rows + row] - mu) * LOG2E);
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) l += __shfl_xor(l, d, 32);
        if (4 * lane < a.D) {
#pragma unroll 4
            for (int s = part; s < a.splits; s += a.share) {
                const float f = exp2_hw((a.pm[s * a.rows + row] - mu) * LOG2E);
                const float4 p = *reinterpret_cast<const float4 *>(a.po + (s * a.rows + row) * a.D + 4 * lane);
                x.x = __builtin_fmaf(p.x, f, x.x);
                x.y = __builtin_fmaf(p.y, f, x.y);
                x.z = __builtin_fmaf(p.z, f, x.z);
                x.w = __builtin_fmaf(p.w, f, x.w);
            }
        }
    }
    if (a.share > 1) {
        sum[grp][lane] = x;
        __syncthreads();
        for (int i = 1; i < a.share && part == 0; ++i) {
            const float4 y = sum[grp + i][lane];
            x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
        }
    }
    if (!row_ok || part) return;
    if (4 * lane < a.D) {
        if (a.out) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            x.x *= inv; x.y *= inv; x.z *= inv; x.w *= inv;
            store4(static_cast<T *>(a.out) + row * a.D + 4 * lane, x.x, x.y, x.z, x.w);
            if (sizeof(T) == 2 && a.rest) *reinterpret_cast<uint32_t *>(a.rest + row * a.D + 4 * lane) = rest4(x.x, x.y, x.z, x.w);
        } else {
            store4(a.so + row * a.D + 4 * lane, x.x, x.y, x.z, x.w);
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

// sums of the splits of a gradient, rounded to the element type (n a multiple of 4); of two gradients for grid.y = 2,
// whose parts follow each other
template <class T>
__global__ void __launch_bounds__(256)
nsd_attn_sum_kernel(const float *part, size_t n, int splits, T *out, T *out2)
{
    const size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (blockIdx.y) { part += splits * n; out = out2; }
    if (i >= n) return;
    float4 x = *reinterpret_cast<const float4 *>(part + i);
#pragma unroll 4
    for (int s = 1; s < splits; ++s) {
        const float4 y = *reinterpret_cast<const float4 *>(part + s * n + i);
        x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
    }
    store4(out + i, x.x, x.y, x.z, x.w);
}

// ---------------------------------------------------------------------
// backward, first part: dQ = scale dS K with dS = P (dP - delta), dP = dO V^T, delta = rowsum(dO O), which it leaves for
// the second part.  Layout of the forward: a wave owns 32 rows, S^T and dP^T are computed from the same tiles.
// ---------------------------------------------------------------------
template <class T, int DP, int WM, int NK, int NBUF>
__global__ void __launch_bounds__(256, sizeof(T) == 2 && 2 * NBUF * 32 * NK * (4 / WM) * DP * 2 <= 81920 ? 2 : 1)
nsd_attn_bwd_q_kernel(SeqArgs a)
{
    constexpr int WN = 4 / WM, BM = 32 * WM, BN = 32 * NK * WN, DT = DP / 32, KC = DP / 16;
    // where workgroups are few and the launch waits on latencies, dS enters its product with 16 bits instead of 8: the
    // error of dQ against 64 bits is then 1.1 instead of 1.4 times that of one rounding, for nothing
    constexpr bool FINE = sizeof(T) == 2 && WM == 1;
    constexpr int NW = BN > 64 ? BN / 64 : 1;
    using TL = Tile<T, DP>;
    constexpr int TB = BN * TL::RB;
    static_assert(WN == 1 || 2 * NBUF * TB >= 4 * 32 * DP * 4, "the waves' sums meet in the tiles' place");
    __shared__ __align__(16) char smem[2 * NBUF * TB];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, c32 = lane & 31;
    const int wm = w % WM, wn = w / WM;
    const int rtiles = (a.R + BM - 1) / BM;
    int pair, tile;
    work_of(blockIdx.x, rtiles, a.Z * a.KVH * a.splits, a.batch, pair, tile);
    const int rt = rtiles - 1 - tile, split = pair % a.splits, kvh = pair / a.splits % a.KVH, z = pair / a.splits / a.KVH;
    const uint8_t *mask = a.mask ? a.mask + (size_t)z * a.Lk : nullptr;
    const int r0 = rt * BM, rho = r0 + wm * 32 + c32;
    const bool row_ok = rho < a.R;
    const int off = a.Lk - a.Lq;
    const int i_row = div_g(row_ok ? rho : a.R - 1, a.g_magic, a.G);
    const int head = kvh * a.G + ((row_ok ? rho : a.R - 1) - i_row * a.G);
    const int last = a.causal ? i_row + off : a.Lk;
    int kend = a.Lk;
    if (a.causal) kend = min(kend, div_g(min(r0 + BM, a.R) - 1, a.g_magic, a.G) + off + 1);
    const int t_end = min((split + 1) * a.split_tiles, kend > 0 ? (kend + BN - 1) / BN : 0);
    int t = split * a.split_tiles;
    const T *kb = static_cast<const T *>(a.k) + z * a.k_sz + kvh * a.k_sh;
    const T *vb = static_cast<const T *>(a.v) + z * a.v_sz + kvh * a.v_sh;
    const size_t row = ((size_t)z * a.Lq + i_row) * (a.KVH * a.G) + head;
    const size_t prow = ((size_t)z * a.KVH + kvh) * a.R + rho;

    constexpr uint64_t PART = BN < 64 ? (1ull << (BN & 63)) - 1 : ~0ull;
    KeyMask<NW> keys{mask, a.Lk, {}};
    if (t < t_end) keys.ask(t * BN);
    Frag<T> qf[KC], gf[KC];
    float delta = 0.0f;
    {
        const T *qp = static_cast<const T *>(a.q) + z * a.q_sz + i_row * a.q_st + head * a.q_sh;
        const T *gp = static_cast<const T *>(a.dout) + row * a.D, *op = static_cast<const T *>(a.out) + row * a.D;
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) {
            qf[kc] = mem_frag(qp, 16 * kc + 8 * h, a.D, row_ok);
            gf[kc] = mem_frag(gp, 16 * kc + 8 * h, a.D, row_ok);
            const Frag<T> of = mem_frag(op, 16 * kc + 8 * h, a.D, row_ok);
            delta = frag_dot(gf[kc], of, delta);
            if (a.rest && row_ok && 16 * kc + 8 * h < a.D) delta = rest_dot(gf[kc], of, a.rest + row * a.D + 16 * kc + 8 * h, delta);
        }
        delta = half_sum(delta);
    }
    if (h == 0 && row_ok && wn == 0 && split == 0) a.delta[prow] = delta;
    const float lse2 = row_ok ? a.lse[prow] * LOG2E : 0.0f;
    f32x16 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[dt][e] = 0.0f;

    // Double buffer: while a tile is worked on, the next one is on its way, and the mask bytes of the one after that.
    uint64_t word[NW], next[NW];
    bool any = false, next_any = false;                         // tiles without a visible key are passed over
    const Stage<T, DP, BN> stage;
    auto fetch = [&](int tile, const char *s) {
        next_any = keys.words(next, PART);
        if (next_any) {
            stage.load(kb + (int64_t)tile * BN * a.k_st, a.k_st, a.D, next, s);
            stage.load(vb + (int64_t)tile * BN * a.v_st, a.v_st, a.D, next, s + TB);
        }
        keys.ask((tile + 1) * BN);
    };
    if (NBUF == 2 && t < t_end) fetch(t, smem);
    for (int buf = 0; t < t_end; ++t, buf ^= NBUF - 1) {
        const char *sk = smem + buf * 2 * TB, *sv = sk + TB;
        if (NBUF == 1) {
            __syncthreads();                                    // everyone has read the last tile
            fetch(t, smem);
        }
        tile_barrier();                                         // the tile is there (and the other buffer free)
        any = next_any;
#pragma unroll
        for (int i = 0; i < NW; ++i) word[i] = next[i];
        if (NBUF == 2 && t + 1 < t_end) fetch(t + 1, smem + (buf ^ 1) * 2 * TB);
        if (!any) continue;
        const int kw0 = wn * 32 * NK, n_vis = last + 1 - (t * BN + kw0);
        uint64_t vis = word[NW > 1 ? kw0 >> 6 : 0] >> (kw0 & 63);
        vis = n_vis <= 0 ? 0 : n_vis < 64 ? vis & ((1ull << n_vis) - 1) : vis;
#pragma unroll
        for (int n = 0; n < NK; ++n) {
            f32x16 s, dp;
#pragma unroll
            for (int e = 0; e < 16; ++e) { s[e] = 0.0f; dp[e] = -delta; }
#pragma unroll
            for (int kc = 0; kc < KC; ++kc) {
                mma(s, TL::row_frag(sk, kw0 + 32 * n, kc, lane), qf[kc]);
                mma(dp, TL::row_frag(sv, kw0 + 32 * n, kc, lane), gf[kc]);
            }
            if constexpr (sizeof(T) == 2) feed<2 * KC, 1, 4>();
            const uint32_t bits = (uint32_t)(vis >> (32 * n)) >> (4 * h);
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = exp2_hw(__builtin_fmaf(s[e], a.scale2, -lse2)) * dp[e];
            if (__ballot((uint32_t)(vis >> (32 * n)) != 0xffffffffu) != 0) {        // (605 -> 576 us for one sequence of 8192)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = bits >> (8 * (e >> 2) + (e & 3)) & 1 ? s[e] : 0.0f;
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const Frag<T> p = acc_frag(s, c, T{}), rest = rest_frag(s, c, p);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    const Frag<T> k = TL::col_frag(sk, kw0 + 32 * n + 16 * c, dt, lane);
                    mma(o[dt], k, p);
                    if constexpr (FINE) mma(o[dt], k, rest);
                }
            }
            if constexpr (sizeof(T) == 2 && !FINE) feed<2 * DT, 2, 4>();
        }
    }
    if constexpr (WN > 1) {                                     // the sums of a row's waves meet
        float *js = reinterpret_cast<float *>(smem);
        __syncthreads();
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                js[(w * DP + 32 * dt + 8 * (e >> 2) + 4 * h + (e & 3)) * 32 + c32] = o[dt][e];
        __syncthreads();
        if (wn) return;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e)
#pragma unroll
                for (int i = 1; i < WN; ++i)
                    o[dt][e] += js[((wm + i * WM) * DP + 32 * dt + 8 * (e >> 2) + 4 * h + (e & 3)) * 32 + c32];
    }
    if (a.splits > 1) {
        float *pp = row_ok ? a.part + ((size_t)split * a.Z * a.Lq * (a.KVH * a.G) + row) * a.D : nullptr;
        put_rows<float, DP>(nullptr, o, a.scale, a.D, lane, [&](int) { return pp; });
        return;
    }
    if (WN == 1) __syncthreads();                               // everyone is done with the tiles
    put_rows<T, DP>(smem + wm * (WN > 1 ? 32 * DP * 4 : 32 * (DP * 2 + 16)), o, a.scale, a.D, lane, [&](int r) {
        const int x = r0 + wm * 32 + r, i = div_g(x, a.g_magic, a.G);
        return x < a.R ? static_cast<T *>(a.dq) + ((((size_t)z * a.Lq + i) * a.KVH + kvh) * a.G + (x - i * a.G)) * a.D : nullptr;
    });
}

// ---------------------------------------------------------------------
// backward, second part: dV = P^T dO, dK = scale dS^T Q.  A wave owns 32 keys, whose K and V stay in its registers, and
// walks over the rows of all G heads (their gradients of a shared head add up in the accumulators): S = Q K^T and
// dP = dO V^T with a lane per key, so that P and dS lie as the B operands of dV^T = dO^T P and dK^T = Q^T dS.  Of a
// workgroup's waves WK lie along the keys and WR = 4 / WK share the rows of a tile, NS sub-tiles of 32 each; their sums
// meet at the end.  Rows are walked from the last one, which all keys see: the workgroups of a kv head then read the same
// rows at the same time.
// ---------------------------------------------------------------------
template <class T, int DP, int WK, int NS, int NBUF>
__global__ void __launch_bounds__(256, sizeof(T) == 2 && 2 * NBUF * 32 * NS * (4 / WK) * DP * 2 <= 81920 ? 2 : 1)
nsd_attn_bwd_kv_kernel(SeqArgs a)
{
    constexpr int WR = 4 / WK, BN = 32 * WK, BM = 32 * WR * NS, DT = DP / 32, KC = DP / 16;
    constexpr bool FINE = sizeof(T) == 2 && WK == 1;            // as in the first part
    using TL = Tile<T, DP>;
    constexpr int TB = BM * TL::RB;
    static_assert(WR == 1 || 2 * NBUF * TB >= 4 * 32 * DP * 4, "the waves' sums meet in the tiles' place");
    __shared__ __align__(16) char smem[2 * NBUF * TB];
    __shared__ __align__(16) float stat[NBUF][2][BM];
    __shared__ int unseen[NBUF][BM / 64];                       // whether a tile has rows that saw no key, of 64 each
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, c32 = lane & 31;
    const int wk = w % WK, wr = w / WK;
    int pair, kt;                                               // the first keys are seen by most rows
    work_of(blockIdx.x, (a.Lk + BN - 1) / BN, a.Z * a.KVH * a.splits, a.batch, pair, kt);
    const int split = pair % a.splits, kvh = pair / a.splits % a.KVH, z = pair / a.splits / a.KVH;
    const int j = kt * BN + wk * 32 + c32;
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
    const int t_last = (a.R + BM - 1) / BM - 1;
    int t_first = lo0 > 0 ? (int)min(lo0 / BM, (int64_t)t_last + 1) : 0, t = t_last;
    if (a.splits > 1) {                                         // this split's part of the rows that see these keys
        const int n = (t_last + 1 - t_first + a.splits - 1) / a.splits;
        t -= split * n;
        t_first = max(t_first, t - n + 1);
    }
    if (a.mask && !__syncthreads_or(key_ok)) t_first = t + 1;   // keys that nobody sees

    f32x16 dk[DT], dv[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) { dk[dt][e] = 0.0f; dv[dt][e] = 0.0f; }

    float st_l = 0.0f, st_d = 0.0f;
    const size_t pbase = ((size_t)z * a.KVH + kvh) * a.R;
    const T *qb = static_cast<const T *>(a.q) + z * a.q_sz, *gb = static_cast<const T *>(a.dout) + (size_t)z * a.Lq * (a.KVH * a.G) * a.D;
    const Stage<T, DP, BM> stage;
    auto fetch = [&](int tile, const char *sm) {
        const uint32_t dst = lds_at(sm);
#pragma unroll
        for (int u = 0; u < stage.U; ++u) {
            const int r = tile * BM + stage.chunk_row(u) + stage.row, e = stage.chunk_elem(u) + stage.elem;
            const bool ok = r < a.R && e < a.D;
            const int tok = div_g(r, a.g_magic, a.G), hd = kvh * a.G + r - tok * a.G;
            const uint64_t zero = (uint64_t)zero_page;
            to_lds(ok ? (uint64_t)(qb + tok * a.q_st + hd * a.q_sh + e) : zero, stage.place(dst, u));
            to_lds(ok ? (uint64_t)(gb + ((size_t)tok * (a.KVH * a.G) + hd) * a.D + e) : zero, stage.place(dst + TB, u));
        }
        if (threadIdx.x < BM) {
            const int r = tile * BM + (int)threadIdx.x;
            st_l = r < a.R ? a.lse[pbase + r] * LOG2E : __builtin_inff();       // no row: probability 0
            st_d = r < a.R ? a.delta[pbase + r] : 0.0f;
        }
    };
    auto put_stat = [&](int b) {
        if (threadIdx.x < BM) {
            stat[b][0][threadIdx.x] = st_l;
            stat[b][1][threadIdx.x] = st_d;
            unseen[b][threadIdx.x >> 6] = __ballot(st_l == -__builtin_inff()) != 0;
        }
    };
    // A row that saw no key has part in nothing, so what its query and its gradient hold (the padding in front of a
    // sequence) may be NaN, which 0 * NaN would spread over dK and dV: zeros instead.  (In the tile, once it is there: left
    // out while it is fetched, by the log-sums of a tile before, the kernel spills and the tiles wait for those.  The question
    // takes 1 of 88 us at 8 x 640 positions.)
    auto blank = [&](int b, char *sq, char *sg) {
        for (int i = threadIdx.x; i < TB / 16; i += 256)
            if (stat[b][0][i / 64 / TL::CG * 16 + (i & 63) / 4] == -__builtin_inff())
                *reinterpret_cast<uint4 *>(sq + i * 16) = *reinterpret_cast<uint4 *>(sg + i * 16) = make_uint4(0, 0, 0, 0);
        __syncthreads();
    };
    if (NBUF == 2 && t >= t_first) {
        fetch(t, smem);
        put_stat(0);
    }
    for (int buf = 0; t >= t_first; --t, buf ^= NBUF - 1) {
        char *sq = smem + buf * 2 * TB, *sg = sq + TB;
        if (NBUF == 1) {
            __syncthreads();                                    // everyone has read the last tile
            fetch(t, smem);
            put_stat(0);
        }
        tile_barrier();
        if (NBUF == 2 && t > t_first) fetch(t - 1, smem + (buf ^ 1) * 2 * TB);
        if (a.mask || off < 0) {                                // (else every row sees a key)
            int none = 0;
#pragma unroll
            for (int i = 0; i < BM / 64; ++i) none |= unseen[buf][i];
            if (__builtin_amdgcn_readfirstlane(none)) blank(buf, sq, sg);
        }
#pragma unroll 1
        for (int i = 0; i < NS; ++i) {
            const int n = wr + WR * i;
            const int thr = first - (t * BM + 32 * n + 4 * h);
            f32x16 s, dp;
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = 0.0f;
#pragma unroll
            for (int kc = 0; kc < KC; ++kc) mma(s, TL::row_frag(sq, 32 * n, kc, lane), kf[kc]);
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const float4 x = *reinterpret_cast<const float4 *>(&stat[buf][1][32 * n + 8 * b + 4 * h]);
                dp[4 * b] = -x.x; dp[4 * b + 1] = -x.y; dp[4 * b + 2] = -x.z; dp[4 * b + 3] = -x.w;
            }
#pragma unroll
            for (int kc = 0; kc < KC; ++kc) mma(dp, TL::row_frag(sg, 32 * n, kc, lane), vf[kc]);
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const float4 x = *reinterpret_cast<const float4 *>(&stat[buf][0][32 * n + 8 * b + 4 * h]);
                const float ls[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float p = exp2_hw(__builtin_fmaf(s[4 * b + e], a.scale2, -ls[e]));
                    s[4 * b + e] = 8 * b + e >= thr ? p : 0.0f;
                }
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) dp[e] = s[e] != 0.0f ? s[e] * dp[e] : 0.0f;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const Frag<T> p = acc_frag(s, c, T{}), ds = acc_frag(dp, c, T{});
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    mma(dv[dt], TL::col_frag(sg, 32 * n + 16 * c, dt, lane), p);
                    mma(dk[dt], TL::col_frag(sq, 32 * n + 16 * c, dt, lane), ds);
                }
                if constexpr (FINE) {
                    const Frag<T> p_rest = rest_frag(s, c, p), ds_rest = rest_frag(dp, c, ds);
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) {
                        mma(dv[dt], TL::col_frag(sg, 32 * n + 16 * c, dt, lane), p_rest);
                        mma(dk[dt], TL::col_frag(sq, 32 * n + 16 * c, dt, lane), ds_rest);
                    }
                }
            }
        }
        if (NBUF == 2 && t > t_first) put_stat(buf ^ 1);
    }
    if constexpr (WR > 1) {
        float *js = reinterpret_cast<float *>(smem);
        f32x16 *acc[2] = {dk, dv};
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            __syncthreads();
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    js[(w * DP + 32 * dt + 8 * (e >> 2) + 4 * h + (e & 3)) * 32 + c32] = acc[x][dt][e];
            __syncthreads();
            if (wr == 0) {
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
#pragma unroll
                        for (int i = 1; i < WR; ++i)
                            acc[x][dt][e] += js[((wk + i * WK) * DP + 32 * dt + 8 * (e >> 2) + 4 * h + (e & 3)) * 32 + c32];
            }
        }
        if (wr) return;
    }
    if (!key_ok) {                                              // a masked key has no part in anything
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) { dk[dt][e] = 0.0f; dv[dt][e] = 0.0f; }
    }
    const size_t all = (size_t)a.Z * a.Lk * a.KVH * a.D;
    auto place = [&](int r) {                                   // of key r of the wave's 32, in elements; -1: no key
        const int x = kt * BN + wk * 32 + r;
        return x < a.Lk ? (int64_t)((((size_t)z * a.Lk + x) * a.KVH + kvh) * a.D) : -1;
    };
    if (a.splits > 1) {
        const int64_t x = place(c32);
        put_rows<float, DP>(nullptr, dk, a.scale, a.D, lane, [&](int) { return x < 0 ? nullptr : a.part + split * all + x; });
        put_rows<float, DP>(nullptr, dv, 1.0f, a.D, lane, [&](int) { return x < 0 ? nullptr : a.part_v + split * all + x; });
        return;
    }
    char *mine = smem + wk * 32 * DP * 4;                       // (what only this wave has read)
    put_rows<T, DP>(mine, dk, a.scale, a.D, lane, [&](int r) { const int64_t x = place(r); return x < 0 ? nullptr : static_cast<T *>(a.dk) + x; });
    put_rows<T, DP>(mine, dv, 1.0f, a.D, lane, [&](int r) { const int64_t x = place(r); return x < 0 ? nullptr : static_cast<T *>(a.dv) + x; });
}

// ---------------------------------------------------------------------
// launchers
// ---------------------------------------------------------------------
constexpr int CUS = 256;
constexpr int64_t MAX_WGS = (1 << 24) - 1;                      // of 256 threads: a launch counts its threads in 32 bits

struct Plan { int wave_rows, bn, tiles, splits, split_tiles; };

int dp_of(int D) { return D <= 64 ? 64 : 128; }
int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Backward: how often the walk over `steps` tiles is split so that `room` workgroups are on the card: whole shares, as a few more
// workgroups than there is room for cost a second round; no share shorter than `least`, below which the join costs more
// than the split gives.
void split_walk(Plan &p, int64_t wgs, int64_t steps, int64_t room, int64_t least)
{
    int64_t s = wgs > 0 ? room / wgs : 1;
    s = s > steps / least ? steps / least : s;
    p.split_tiles = (int)(s > 1 ? div_up(steps, s) : steps > 0 ? steps : 1);
    p.splits = (int)(s > 1 ? div_up(steps, p.split_tiles) : 1);
}

// Forward: the split with the least of (tiles of a share) x (time of a tile) + (time of the join).  In ns, with keys that
// come from memory as a decode's do (another layer's lie between two steps): a bf16 tile takes 1330 and 1950 (head
// dimensions up to 64 and 128; 1600 with few rows) whether one workgroup waits for it on a CU or two, an fp32 tile 3100
// and 5200, with two workgroups 1.5 and 2 times that; the join takes 3 us and 33 ns for each share of 128 rows.  A beam step
// over one prefix, 8 kv heads, as many workgroups as there is room for against this: 1024 hypotheses, 24 heads of 128: 512
// positions 55 and 44 us, 2048 77 and 77, 8192 170 and 171 (2048 without a split: 91); 512 with 16 heads of 64: 37 and 25,
// 41 and 37, 56 and 56.
void split_keys(Plan &p, int64_t wgs, int64_t steps, int DP, int dtype)
{
    const bool wide = DP == 128;
    const int64_t tile = dtype == 0 ? (wide ? 5200 : 3100) : p.wave_rows < 4 ? 1600 : wide ? 1950 : 1330;
    const int64_t pair = dtype == 0 ? (wide ? 200 : 150) : 100;  // percent
    int64_t best = 1, least = steps * tile;
    for (int64_t s = 2; s <= steps && s * wgs <= 2 * CUS; ++s) {
        const int64_t share = div_up(steps, s);
        const int64_t t = share * tile * (s * wgs > CUS ? pair : 100) / 100 + 3000 + s * wgs * p.wave_rows * 33 / 4;
        if (t < least) { least = t; best = s; }
    }
    p.split_tiles = (int)(best > 1 ? div_up(steps, best) : steps > 0 ? steps : 1);
    p.splits = (int)(best > 1 ? div_up(steps, p.split_tiles) : 1);
}

// Forward: row tiles of 128 (four waves along the rows) unless there are at most 64 or 32 rows: the waves then share the
// keys of a tile.  (Tiles of 64 rows where they would fit the rows better, 189 of them for instance, take longer: 76
// against 61 us for 96 x 63 queries over 320 keys; as do tiles of 32 keys with three waves per SIMD, whose registers
// spill: 484 against 442 us for one sequence of 8192.)
Plan fwd_plan(int Z, int KVH, int R, int Lk, int D, int dtype)
{
    Plan p;
    p.wave_rows = R <= 32 ? 1 : R <= 64 ? 2 : 4;
    p.bn = (dtype == 0 || p.wave_rows < 4 ? 32 : 64) * (4 / p.wave_rows);
    p.tiles = (int)div_up(R, 32 * p.wave_rows);
    split_keys(p, (int64_t)p.tiles * KVH * Z, div_up(Lk, p.bn), dp_of(D), dtype);
    return p;
}

// Backward, dQ: 128 rows where that makes a workgroup for every CU, else 64 or 32 (the waves share the keys): fp32, 3 x 217
// positions of 6 heads, 51 us with 128 rows, 27 with 32, 21 with the keys split as well.  (tests/test_seq_ops_range.py restates
// this choice and bwd_kv_plan's to reach every form.)
Plan bwd_q_plan(int Z, int KVH, int R, int Lk, int D, int dtype)
{
    Plan p;
    const int64_t pairs = (int64_t)Z * KVH;
    p.wave_rows = R > 64 && pairs * div_up(R, 128) >= CUS ? 4 : R > 32 && pairs * div_up(R, 64) >= CUS ? 2 : 1;
    p.bn = p.wave_rows == 4 ? (dtype == 0 && dp_of(D) == 128 ? 32 : 64) : 32 * (4 / p.wave_rows);
    p.tiles = (int)div_up(R, 32 * p.wave_rows);
    split_walk(p, p.tiles * pairs, div_up(Lk, p.bn), CUS, dtype == 0 ? 1 : 8);
    return p;
}

// Backward, dK and dV: 64 keys (two waves along the keys, two along the rows), or 32 where that leaves CUs without work.
// Four waves along the keys, 128 of them, are slower: 119 against 86 us at 8 x 640 positions, 1439 against 1014 us at one
// sequence of 8192 (24 query heads, 8 kv heads of 128): half as many workgroups, and unequal ones under a causal mask.
Plan bwd_kv_plan(int Z, int KVH, int R, int Lk, int D, int dtype)
{
    Plan p;
    const int64_t pairs = (int64_t)Z * KVH;
    p.wave_rows = Lk > 32 && pairs * div_up(Lk, 64) >= CUS / 2 ? 2 : 1;     // (waves along the keys here)
    p.bn = 32 * p.wave_rows;
    p.tiles = (int)div_up(Lk, p.bn);
    split_walk(p, p.tiles * pairs, div_up(R, 32 * (4 / p.wave_rows)), CUS, dtype == 0 ? 1 : 8);
    return p;
}

// pairs of an XCD that are worked on together: two rounds of its 64 workgroups
int pair_batch(int64_t pairs, int64_t tiles)
{
    const int64_t per = pairs % 8 == 0 ? pairs / 8 : pairs, b = pairs % 8 == 0 ? 128 / tiles : per;
    return (int)(b < 1 ? 1 : b > per ? per : b);
}

dim3 grid_of(SeqArgs &a, const Plan &p)
{
    const int64_t pairs = (int64_t)a.KVH * a.Z * p.splits;
    a.splits = p.splits;
    a.split_tiles = p.split_tiles;
    a.batch = pair_batch(pairs, p.tiles);
    return dim3((unsigned)(p.tiles * pairs));
}

template <class T, int DP, bool STATE>
void launch_fwd(SeqArgs a, const Plan &p, hipStream_t s)
{
    constexpr bool F = sizeof(T) == 4;
    const dim3 grid = grid_of(a, p), block(256);
    if (p.wave_rows == 4) hipLaunchKernelGGL((nsd_attn_fwd_kernel<T, DP, 4, F ? 32 : 64, 2, STATE>), grid, block, 0, s, a);
    else if (p.wave_rows == 2) hipLaunchKernelGGL((nsd_attn_fwd_kernel<T, DP, 2, 32, 2, STATE>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((nsd_attn_fwd_kernel<T, DP, 1, 32, F && DP == 128 ? 1 : 2, STATE>), grid, block, 0, s, a);
}

int run_join(JoinArgs j, int dtype, hipStream_t s)
{
    j.share = j.splits >= 8 ? 8 : j.splits >= 4 ? 4 : 2;
    const dim3 grid((unsigned)((j.rows * j.share + 7) / 8)), block(256);
    if (dtype == 0) hipLaunchKernelGGL(nsd_attn_join_kernel<float>, grid, block, 0, s, j);
    else hipLaunchKernelGGL(nsd_attn_join_kernel<BF16>, grid, block, 0, s, j);
    return (int)hipGetLastError();
}

template <bool STATE>
int run_fwd(const SeqArgs &a, const Plan &p, int dtype, hipStream_t s)
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

template <class T>
void launch_sum(const float *part, size_t n, int splits, void *out, void *out2, hipStream_t s)
{
    hipLaunchKernelGGL(nsd_attn_sum_kernel<T>, dim3((unsigned)((n + 1023) / 1024), out2 ? 2 : 1), dim3(256), 0, s, part, n, splits, (T *)out,
                       (T *)out2);
}

// Scratch of the backward pass: the rows' delta, then the parts of dQ, and in the same place those of dK and dV.
struct BwdScratch { size_t delta, q, kv; };
BwdScratch bwd_scratch(const Plan &q, const Plan &kv, size_t rows, size_t keys, size_t D)
{
    return {(rows + 3) / 4 * 16, q.splits > 1 ? q.splits * rows * D * 4 : 0, kv.splits > 1 ? 2 * kv.splits * keys * D * 4 : 0};
}

template <class T, int DP>
void launch_bwd(SeqArgs a, const Plan &q, const Plan &kv, hipStream_t s)
{
    constexpr bool F = sizeof(T) == 4, F128 = F && DP == 128;
    const dim3 block(256);
    const size_t nq = (size_t)a.Z * a.Lq * a.KVH * a.G * a.D, nk = (size_t)a.Z * a.Lk * a.KVH * a.D;
    if (a.R > 0) {
        const dim3 grid = grid_of(a, q);
        if (q.wave_rows == 4) hipLaunchKernelGGL((nsd_attn_bwd_q_kernel<T, DP, 4, F128 ? 1 : 2, 2>), grid, block, 0, s, a);
        else if (q.wave_rows == 2) hipLaunchKernelGGL((nsd_attn_bwd_q_kernel<T, DP, 2, 1, 2>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((nsd_attn_bwd_q_kernel<T, DP, 1, 1, F128 ? 1 : 2>), grid, block, 0, s, a);
        if (q.splits > 1) launch_sum<T>(a.part, nq, q.splits, a.dq, nullptr, s);
    }
    if (a.Lk > 0) {
        const dim3 grid = grid_of(a, kv);
        a.part_v = a.part + kv.splits * nk;
        if (kv.wave_rows == 2) hipLaunchKernelGGL((nsd_attn_bwd_kv_kernel<T, DP, 2, 1, 2>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((nsd_attn_bwd_kv_kernel<T, DP, 1, 1, F128 ? 1 : 2>), grid, block, 0, s, a);
        if (kv.splits > 1) launch_sum<T>(a.part, nk, kv.splits, a.dk, a.dv, s);
    }
}

bool al16(const void *p) { return ((uintptr_t)p & 15u) == 0; }

// the shape fields that the entry points share
int shape_check(const NsdSeqAttn *p)
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
    if (zk > (1ll << 30) || zk * ((R + 31) / 32) > (1ll << 30) || zk * (((int64_t)p->len_k + 31) / 32) > (1ll << 30)) return NSD_E_SIZE;
    if (zk * div_up(R, R <= 32 ? 32 : R <= 64 ? 64 : 128) > MAX_WGS) return NSD_E_SIZE;    // (the tiles of many rows)
    return NSD_OK;
}

int bwd_shape_check(const NsdSeqAttn *p)
{
    if (const int rc = shape_check(p)) return rc;
    if (p->key_len) return NSD_E_SIZE;                          // ragged keys are a form of the prefix state only
    return (int64_t)p->batch * p->kv_heads * div_up(p->len_k, p->len_k <= 32 ? 32 : 64) > MAX_WGS ? NSD_E_SIZE : NSD_OK;
}

// the same as kernel arguments, with the pointers and strides checked (in pieces of 16 bytes)
int seq_args(const NsdSeqAttn *p, const void *q, const void *k, const void *v, SeqArgs &a)
{
    if (const int rc = shape_check(p)) return rc;
    if (p->batch == 0) return NSD_OK;
    const int64_t G = p->heads / p->kv_heads, R = (int64_t)p->len_q * G;
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
    if (shape_check(p) || p->batch == 0 || p->len_q == 0) return 0;
    const int G = p->heads / p->kv_heads;
    const Plan f = fwd_plan(p->batch, p->kv_heads, p->len_q * G, p->len_k, p->hd, p->dtype);
    return f.splits > 1 ? (int64_t)f.splits * p->batch * p->len_q * p->heads * (p->hd + 2) * 4 : 0;
}

extern "C" int nsd_attn_fwd(const void *q, const void *k, const void *v, const NsdSeqAttn *p, void *out, float *lse, uint8_t *rest,
                            void *ws, int64_t ws_bytes, void *stream)
{
    SeqArgs a;
    if (const int rc = seq_args(p, q, k, v, a)) return rc;
    if (p->batch == 0 || p->len_q == 0) return NSD_OK;
    if (!out) return NSD_E_NULL;
    if (!al16(out) || !al16(rest) || !al16(ws)) return NSD_E_ALIGN;
    const Plan f = fwd_plan(a.Z, a.KVH, a.R, a.Lk, a.D, p->dtype);
    a.out = out;
    a.lse = lse;
    a.rest = rest;
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
    JoinArgs j{a.po, a.pm, a.pl, f.splits, a.D, a.KVH, a.G, a.Lq, 0, (size_t)a.Z * a.Lq * a.KVH * a.G, nullptr, nullptr, nullptr, out, rest, lse};
    return run_join(j, p->dtype, (hipStream_t)stream);
}

extern "C" int64_t nsd_attn_bwd_workspace(const NsdSeqAttn *p)
{
    if (bwd_shape_check(p) || p->batch == 0) return 0;
    const int R = p->len_q * (p->heads / p->kv_heads);
    const BwdScratch b = bwd_scratch(bwd_q_plan(p->batch, p->kv_heads, R, p->len_k, p->hd, p->dtype),
                                     bwd_kv_plan(p->batch, p->kv_heads, R, p->len_k, p->hd, p->dtype),
                                     (size_t)p->batch * p->len_q * p->heads, (size_t)p->batch * p->len_k * p->kv_heads, p->hd);
    return (int64_t)(b.delta + (b.q > b.kv ? b.q : b.kv));
}

extern "C" int nsd_attn_bwd(const void *q, const void *k, const void *v, const void *out, const float *lse, const uint8_t *rest,
                            const void *dout, const NsdSeqAttn *p, void *dq, void *dk, void *dv, void *ws, int64_t ws_bytes,
                            void *stream)
{
    SeqArgs a;
    if (const int rc = bwd_shape_check(p)) return rc;
    if (const int rc = seq_args(p, q, k, v, a)) return rc;
    if (p->batch == 0) return NSD_OK;
    if (a.R > 0 && (!out || !lse || !dout || !dq || !ws)) return NSD_E_NULL;
    if (a.Lk > 0 && (!dk || !dv)) return NSD_E_NULL;
    if (!al16(out) || !al16(rest) || !al16(dout) || !al16(dq) || !al16(dk) || !al16(dv) || !al16(ws)) return NSD_E_ALIGN;
    const Plan pq = bwd_q_plan(a.Z, a.KVH, a.R, a.Lk, a.D, p->dtype), pk = bwd_kv_plan(a.Z, a.KVH, a.R, a.Lk, a.D, p->dtype);
    const BwdScratch b = bwd_scratch(pq, pk, (size_t)a.Z * a.KVH * a.R, (size_t)a.Z * a.KVH * a.Lk, a.D);
    if (ws_bytes < (int64_t)(b.delta + (b.q > b.kv ? b.q : b.kv))) return NSD_E_SIZE;
    a.out = const_cast<void *>(out);
    a.lse = const_cast<float *>(lse);
    a.rest = const_cast<uint8_t *>(rest);
    a.dout = dout;
    a.delta = (float *)ws;
    a.part = (float *)((char *)ws + b.delta);
    a.dq = dq; a.dk = dk; a.dv = dv;
    if (p->dtype == 0) {
        if (dp_of(a.D) == 64) launch_bwd<float, 64>(a, pq, pk, (hipStream_t)stream);
        else launch_bwd<float, 128>(a, pq, pk, (hipStream_t)stream);
    } else {
        if (dp_of(a.D) == 64) launch_bwd<BF16, 64>(a, pq, pk, (hipStream_t)stream);
        else launch_bwd<BF16, 128>(a, pq, pk, (hipStream_t)stream);
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
    const Plan f = fwd_plan(a.Z, a.KVH, a.R, a.Lk, a.D, p->dtype);
    const size_t rows = (size_t)a.Z * a.Lq * a.KVH * a.G;
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
    JoinArgs j{a.po, a.pm, a.pl, f.splits, a.D, a.KVH, a.G, a.Lq, 0, rows, part_o, part_m, part_l, nullptr, nullptr, nullptr};
    return run_join(j, p->dtype, (hipStream_t)stream);
}
