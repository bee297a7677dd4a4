// Attention over the paged 4-bit KV cache (kvcache4.h): the mathematics, row blocks,
// pieces and running softmax of attnp.h, over values code * sub * scale.
//
// code * sub is a whole number up to 1016 in magnitude and exact in f16, so the matrix
// cores get it as one operand, and the f32 operand split into two f16 numbers as
// for the 8-bit cache: results are of f32 accuracy. A nibble n (a code plus 8) is a subnormal
// f16 number where it lies, and one packed FMA, n sub - 8 sub, makes the product of two
// without a rounding: nine instructions for eight values (the bytes of the 8-bit cache take ten). What is left of a key's and a
// value's scale is one factor a token: scores are multiplied by the key's, weights by the
// value's before they are split.
#pragma once

#include <limits.h>

#include "attnp.h"
#include "kvcache4.h"

namespace sihip {

// C: of the cache, with codes in place of bytes and no scales
struct Attn4Args : AttnPArgs {
    const int8_t *ksub, *vsub;
    const uint16_t *kd, *vd;
};

typedef uint32_t ap_u4 __attribute__((ext_vector_type(4)));

// Products are in units of 2^-16: a nibble n where it lies in a half word, at bit 0 or 4, is the
// f16 number n 2^-24 or n 2^-20 (subnormal, which costs the packed FMA nothing). Elements 0, 1
// and 4, 5 of a word are at bit 0 of their halves (the latter after a shift by 8), 2, 3 and 6, 7 at bit 4.
constexpr int kAp4Bits = 16;
constexpr float kAp4Unit = 1 << kAp4Bits;

// subs of a pair of elements: times 2^8 or 2^4, which any byte allows (2^9 times -128, of memory
// that was never written, would be infinite), and -8 sub 2^-16
struct Ap4Sub {
    ap_h2 lo, m;
};

// eight nibbles times the subs of their elements, s[i] of elements 2 i and 2 i + 1
__device__ inline ap_h8 ap4_cvt(uint32_t w, const Ap4Sub (&s)[4]) {
    union {
        ap_h8 v;
        ap_h2 h[4];
    } u;
    const uint32_t n[4] = {w & 0x000f000fu, w & 0x00f000f0u, w >> 8 & 0x000f000fu, w >> 8 & 0x00f000f0u};
#pragma unroll
    for (int i = 0; i < 4; i++) u.h[i] = __builtin_elementwise_fma(__builtin_bit_cast(ap_h2, n[i]), s[i].lo, s[i].m);
    return u.v;
}

// a pair of subs for pair i of a word
__device__ inline Ap4Sub ap4_scaled(ap_h2 sub, int i) {
    const _Float16 f = (_Float16)(i & 1 ? 0x1p4f : 0x1p8f), g = (_Float16)-0x1p-13f;
    return {sub * ap_h2{f, f}, sub * ap_h2{g, g}};
}

// byte t of x (a sub) for all elements of a word
__device__ inline void ap4_sub(uint32_t x, int t, Ap4Sub (&s)[4]) {
    const ap_h2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
    const ap_h2 v = __builtin_bit_cast(ap_h2, __builtin_amdgcn_perm(0x64646464u, x ^ 0x80808080u, 0x04000400u | (uint32_t)t * 0x00010001u)) - off;
#pragma unroll
    for (int i = 0; i < 4; i++) s[i] = ap4_scaled(v, i);
}

// the eight bytes of x and y (subs) for the elements of a word
__device__ inline void ap4_subs(uint32_t x, uint32_t y, Ap4Sub (&s)[4]) {
    ap_h2 v[4];
    ap_cvt4(x, v[0], v[1]);
    ap_cvt4(y, v[2], v[3]);
#pragma unroll
    for (int i = 0; i < 4; i++) s[i] = ap4_scaled(v[i], i);
}

// a bfloat16 in the low or high half of x
__device__ inline float ap4_bf16(uint32_t x, int high) { return __builtin_bit_cast(float, high ? x & 0xffff0000u : x << 16); }

// What turns a row's sums of products times a key's scale, in units of 2^-e times its queries' power of two, into scores in
// log2 units (f) or the argument of the tanh (fc). Of large queries f can pass the largest number where scores do not, as keys
// are small; of small ones the sums times a large key's scale can. Where f passes 2^100, or is below 2^least, it is 2^64 less or
// more, and sums are multiplied by what is returned first. (Scores that pass 2^68 on the way have no weights in f32.) f is
// above zero: it leaves -inf as it is.
__device__ inline float ap4_factors(const AttnPArgs &A, int e, int least, float &f, float &fc) {
    const int size = e + __builtin_amdgcn_frexp_expf(A.scale2);
    const bool large = size > 100, small = size < least;
    e += large ? -64 : small ? 64 : 0;
    f = fminf(fmaxf(ldexpf(A.scale2, e), 0x1p-149f), FLT_MAX);
    fc = fminf(ldexpf(A.cap_in, e), FLT_MAX);
    return large ? 0x1p64f : small ? 0x1p-64f : 1.0f;
}

// Chunk u of u0 .. u1 - 1, the nearest first. With slopes scores rise towards a row's own position, and in
// the other order nearly every chunk would move the maximum and the sums with it: 3 prompts of up to 4096, 40 heads, 810
// us and 680 this way; 64 single tokens over up to 8192 73 and 68. Without them both orders take the same.
__device__ inline int ap4_chunk(const Sight &S, int u0, int u1, int u) { return ap_chunk(S, u0 + u1 - 1 - u); }

// ---- few rows ----------------------------------------------------------------------
//
// attnp_rows_kernel (attnp.h) over 4-bit values: 16 rows of one request and KV head, one split of
// its chunks of 16 TT keys, global memory to registers. KD dims of a key are a lane's in each of
// NK slices of 4 KD: 16 bytes, or 8 for heads up to 64. Row m of key tile t is token TT m + t, so
// that a lane's TT subs are neighbours, and its scores, of tokens 4 TT g .., are
// i-major: token TT i + t of them is register (t, i).
//
// Bound by its vector instructions: codes to f16, twice a byte of the cache, and subs for the pairs of a
// word. 16 requests of 4 tokens over up to 8192 keys (32 heads of 128 on 8) 35 us, where its 55 MB would take 12; 4096 rows of 16 heads of
// 256, for which there is no large block, 770 (its doubled products 222); a prompt of 509 tokens, 14 heads of 64 on 2, 11.6, of
// which an empty launch takes 3.5 and two chunks a wave, in turn, most of the rest.
template <int KD, int NK, int ND, int TT, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 2) void attnp4_rows_kernel(Attn4Args A) {
    constexpr int CH = 16 * TT, SEG = 4 * TT, KW = KD / 8, VW = SEG / 8;
    constexpr uint32_t kAll = (1u << SEG) - 1;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    const int hd = A.C.hd, shift = A.C.shift, B = 1 << shift;
    int r, h, tile, split, per;
    int64_t piece;
    Span s;
    if (!ap_rows_place(A, r, h, tile, split, per, piece, s)) return;
    const int32_t *table = A.R.table + (int64_t)r * A.R.max_blocks;
    const int n_tok = min(s.n, A.R.max_q), n_rows = n_tok * A.G;
    if (tile * 16 >= n_rows) return;
    const int t0 = tile * 16 / A.G, t1 = min((tile * 16 + 15) / A.G, n_tok - 1);
    const Sight S = ap_sight(A, r, s, t0, t1);
    const int n_split = ap_splits(A, S.n, per);
    if (split >= n_split) return;
    const int u0 = __builtin_amdgcn_readfirstlane((int)((int64_t)S.n * split / n_split));
    const int u1 = __builtin_amdgcn_readfirstlane((int)((int64_t)S.n * (split + 1) / n_split));
    auto chunk_of = [&](int u) { return ap4_chunk(S, u0, u1, u); };

    // table entries of this lane's key rows, and of its values and scores: loaded a chunk ahead,
    // between its keys and its values, and looked at when they are used (a wait for a load is one for
    // all loads before it)
    const int last_block = max(S.keys - 1, 0) >> shift, n_pages = (int)A.C.n_pages;
    auto first_of = [&](int u, int seg) { return chunk_of(u) * CH + seg * SEG; };
    auto entry_of = [&](int u, int seg) { return table[min(first_of(u, seg) >> shift, last_block)]; };
    auto page_of = [&](int u, int seg, int entry) { return first_of(u, seg) < S.keys && entry >= 0 && entry < n_pages ? entry : -1; };
    int u = u0 + wave, ek = 0, ev = 0, pv = 0;
    if (u < u1) {
        ek = entry_of(u, col >> 2);
        ev = entry_of(u, g);
    }

    // this lane's row
    const int row = min(tile * 16 + col, n_rows - 1);
    const int tok = row / A.G, head = h * A.G + row % A.G;
    const int p = s.p0 + tok;
    const float slope = A.slopes ? A.slopes[head] * kLog2e : 0.0f;
    const float *qrow = A.q + (s.q0 + tok) * A.ldq + (int64_t)head * hd;
    // this lane's dims of a key row; those past hd meet zeros of q
    auto dim_of = [&](int e) { return 4 * KD * e + KD * g; };
    float x[NK][KW][8];
#pragma unroll
    for (int e = 0; e < NK; e++)
#pragma unroll
        for (int y = 0; y < KW; y++) ap_load8(qrow + (dim_of(e) < hd ? dim_of(e) : 0) + 8 * y, A.q_vec, x[e][y]);

    // a chunk starts at a multiple of its length: a lane's place in a page is
    // its own and, in longer pages, the chunk's
    const int groups = hd / 32, kt = TT * col & (B - 1), vt = SEG * g & (B - 1);
    const uint32_t row_bytes = hd / 2, head_bytes = row_bytes << shift;
    const uint8_t *kb = (const uint8_t *)A.C.k + kt * row_bytes, *vb = (const uint8_t *)A.C.v + ((col << shift) + vt) / 2;
    uint32_t kr[TT][NK][KW], vr[ND][VW];
    uint32_t ksub[NK], vsub[ND / 2][SEG / 4], kd[SEG / 2], vd[SEG / 2];
    auto load_keys = [&](int u) {
        const int at = chunk_of(u) * CH & (B - 1), pk = page_of(u, col >> 2, ek);
        pv = page_of(u, g, ev);
        const int64_t ph = (int64_t)max(pk, 0) * A.C.n_kv + h, ps = (int64_t)max(pv, 0) * A.C.n_kv + h;
        const uint8_t *kp = kb + (ph * head_bytes + at * row_bytes);
#pragma unroll
        for (int e = 0; e < NK; e++) {
            const int d = dim_of(e) < hd ? dim_of(e) : 0;
#pragma unroll
            for (int t = 0; t < TT; t++) {
                if constexpr (KW == 4) {
                    const uint4 v = *(const uint4 *)(kp + t * row_bytes + d / 2);
                    kr[t][e][0] = v.x, kr[t][e][1] = v.y, kr[t][e][2] = v.z, kr[t][e][3] = v.w;
                } else {
                    const uint2 v = *(const uint2 *)(kp + t * row_bytes + d / 2);
                    kr[t][e][0] = v.x, kr[t][e][1] = v.y;
                }
            }
            const int8_t *sp = A.ksub + ((ph * groups + d / 32) << shift) + at + kt;
            if constexpr (TT == 4) ksub[e] = *(const uint32_t *)sp;
            else ksub[e] = *(const uint16_t *)sp;
        }
        const ap_u4 *dk = (const ap_u4 *)(A.kd + (ps << shift) + at + vt), *dv = (const ap_u4 *)(A.vd + (ps << shift) + at + vt);
#pragma unroll
        for (int i = 0; i < SEG / 8; i++) {
            const ap_u4 a = dk[i], b = dv[i];
#pragma unroll
            for (int e = 0; e < 4; e++) kd[4 * i + e] = a[e], vd[4 * i + e] = b[e];
        }
    };
    auto load_values = [&](int u) {
        const int at = chunk_of(u) * CH & (B - 1);
        const int64_t ph = (int64_t)max(pv, 0) * A.C.n_kv + h;
        const uint8_t *vp = vb + (ph * head_bytes + at / 2);
        const int8_t *sp = A.vsub + ((ph * groups) << shift) + at + vt;
#pragma unroll
        for (int d = 0; d < ND; d++) {
            const uint8_t *to = vp + (min(16 * d, hd - 16) << shift >> 1);
            if constexpr (VW == 2) {
                const uint2 v = *(const uint2 *)to;
                vr[d][0] = v.x, vr[d][1] = v.y;
            } else {
                vr[d][0] = *(const uint32_t *)to;
            }
        }
#pragma unroll
        for (int i = 0; i < ND / 2; i++) {
            const int8_t *from = sp + (min(i, groups - 1) << shift);
            if constexpr (SEG == 16) {
                const ap_u4 v = *(const ap_u4 *)from;
#pragma unroll
                for (int e = 0; e < 4; e++) vsub[i][e] = v[e];
            } else {
                const uint2 v = *(const uint2 *)from;
                vsub[i][0] = v.x, vsub[i][1] = v.y;
            }
        }
    };
    auto load_entries = [&](int u) {
        ek = entry_of(u, col >> 2);
        ev = entry_of(u, g);
    };
    if (u < u1) {
        load_keys(u);
        load_entries(min(u + WAVES, u1 - 1));
        load_values(u);
    }

    // the query, while the first keys are on their way
    ap_h8 qh[NK][KW], ql[NK][KW];
    float f_row, fc_row, turn;
    {
        // (no scale: zeros, so that a score is zero whatever the key)
        const float sign = A.scale2 > 0.0f ? A.sign : 0.0f;
        float amax = 0.0f;
#pragma unroll
        for (int e = 0; e < NK; e++)
#pragma unroll
            for (int y = 0; y < KW; y++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    x[e][y][j] = dim_of(e) < hd ? x[e][y][j] * sign : 0.0f;
                    amax = fmaxf(amax, fabsf(x[e][y][j]));
                }
        const int e2 = ap_row_exponent(ap_max_quarters(amax));
#pragma unroll
        for (int e = 0; e < NK; e++)
#pragma unroll
            for (int y = 0; y < KW; y++) {
#pragma unroll
                for (int j = 0; j < 8; j++) x[e][y][j] = ldexpf(x[e][y][j], e2);
                ap_split8(x[e][y], qh[e][y], ql[e][y]);
            }
        turn = ap4_factors(A, kAp4Bits - e2, -60, f_row, fc_row);
    }
    const bool turned = __any(turn != 1.0f);
    Running R;
    ap_f4 o[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) o[d] = ap_f4{0, 0, 0, 0};
    for (; u < u1; u += WAVES) {
        const int next = min(u + WAVES, u1 - 1), c = chunk_of(u);
        ap_f4 sc[TT];
#pragma unroll
        for (int t = 0; t < TT; t++) sc[t] = ap_f4{0, 0, 0, 0};
        // (two tiles at a time: a product waits for the one before it of its sum)
#pragma unroll
        for (int e = 0; e < NK; e++)
#pragma unroll
            for (int t = 0; t < TT; t += 2) {
                Ap4Sub sub[2][4];
#pragma unroll
                for (int i = 0; i < 2; i++) ap4_sub(ksub[e], t + i, sub[i]);
#pragma unroll
                for (int y = 0; y < KW; y++) {
                    ap_h8 a[2];
#pragma unroll
                    for (int i = 0; i < 2; i++) a[i] = ap4_cvt(kr[t + i][e][y], sub[i]);
#pragma unroll
                    for (int i = 0; i < 2; i++) sc[t + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[i], qh[e][y], sc[t + i], 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 2; i++) sc[t + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[i], ql[e][y], sc[t + i], 0, 0, 0);
                }
            }
        if (turned) {
#pragma unroll
            for (int t = 0; t < TT; t++) sc[t] *= turn;
        }
        // key i of this lane: j0 + i; its score in log2 units is w[i] * f
        const int j0 = c * CH + g * SEG;
        float w[SEG], vs[SEG], f = f_row;
#pragma unroll
        for (int i = 0; i < SEG; i++) {
            w[i] = sc[i % TT][i / TT] * ap4_bf16(kd[i / 2], i & 1);
            vs[i] = ap4_bf16(vd[i / 2], i & 1);
        }
        const bool here = pv >= 0;
        load_keys(next);
        load_entries(min(next + WAVES, u1 - 1));
        if (A.cap != 0.0f) {
#pragma unroll
            for (int i = 0; i < SEG; i++) w[i] = ap_capped(A, w[i] * f, w[i] * fc_row);
            f = 1.0f;
        }
        if (A.slopes) {
            const float far = (float)(j0 - p);
#pragma unroll
            for (int i = 0; i < SEG; i++) w[i] = fmaf(w[i], f, -slope * fabsf(far + (float)i));
            f = 1.0f;
        }
        if (!ap_whole(A, S, c * CH, CH) || __any(!here)) {
            // (what was never written may have any scale)
            const uint32_t hidden = here ? ap_hidden(A, S, p, j0) & kAll : kAll;
#pragma unroll
            for (int i = 0; i < SEG; i++) {
                w[i] = ap_hide(w[i], hidden, i);
                vs[i] = hidden >> i & 1 ? 0.0f : vs[i];
            }
        }
        float mx = w[0];
#pragma unroll
        for (int i = 1; i < SEG; i++) mx = fmaxf(mx, w[i]);
        mx *= f;
        if (__any(mx > R.m + kApLate)) {
            const float ao = R.refer(R.raise(ap_max_quarters(mx)), 0.0f);
#pragma unroll
            for (int d = 0; d < ND; d++) o[d] *= ao;
        }
        // weights, and their products with the values' scales
        float z[SEG], most = 0.0f, few = 0.0f;
#pragma unroll
        for (int i = 0; i < SEG; i++) {
            const float x = __builtin_amdgcn_exp2f(fmaf(w[i], f, -R.m));
            few += x;
            z[i] = x * vs[i];
            most = fmaxf(most, z[i]);
        }
        R.l += few;
        if (__any(most > 16.0f * R.ref)) {
            const float ao = R.refer(1.0f, ap_max_quarters(most));
#pragma unroll
            for (int d = 0; d < ND; d++) o[d] *= ao;
        }
        ap_h8 ph[VW], pl[VW];
#pragma unroll
        for (int e = 0; e < VW; e++) ap_split8w(z + 8 * e, R.over, ph[e], pl[e]);
#pragma unroll
        for (int d = 0; d < ND; d += 2) {
            Ap4Sub sub[VW][4];
#pragma unroll
            for (int e = 0; e < VW; e++) ap4_subs(vsub[d / 2][2 * e], vsub[d / 2][2 * e + 1], sub[e]);
#pragma unroll
            for (int e = 0; e < VW; e++) {
                const ap_h8 a = ap4_cvt(vr[d][e], sub[e]), b = ap4_cvt(vr[d + 1][e], sub[e]);
                o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ph[e], o[d], 0, 0, 0);
                o[d + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b, ph[e], o[d + 1], 0, 0, 0);
                o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pl[e], o[d], 0, 0, 0);
                o[d + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b, pl[e], o[d + 1], 0, 0, 0);
            }
        }
        load_values(next);
    }
    ap_rows_end<ND, WAVES>(A, s, R, o, kAp4Unit / kApUnit, h, tile, n_rows, piece, split, n_split, tok, head);
}

// Codes alone, in units of 2^-10: of a nibble n 2^-24 or n 2^-20 (ap4_cvt) one packed FMA with
// constants. (In units of 2^-24 they would need no factor at bit 0. But they are subnormal then, and the matrix cores add products
// of such numbers with fewer bits: results were off by 10^-5.)
constexpr int kAp4CodeBits = 10;
constexpr float kAp4Code = 1 << kAp4CodeBits;

__device__ inline ap_h8 ap4_codes(uint32_t w) {
    const _Float16 f = (_Float16)0x1p14f, g = (_Float16)0x1p10f, off = (_Float16)-0x1p-7f;
    const ap_h2 scale[2] = {{f, f}, {g, g}}, minus8 = {off, off};
    union {
        ap_h8 v;
        ap_h2 h[4];
    } u;
    const uint32_t n[4] = {w & 0x000f000fu, w & 0x00f000f0u, w >> 8 & 0x000f000fu, w >> 8 & 0x00f000f0u};
#pragma unroll
    for (int i = 0; i < 4; i++) u.h[i] = __builtin_elementwise_fma(__builtin_bit_cast(ap_h2, n[i]), scale[i & 1], minus8);
    return u.v;
}

// signed byte t of x
__device__ inline float ap4_byte(uint32_t x, int t) { return (float)(int8_t)(x >> (8 * t)); }

// the sums of N numbers of a row over its NG columns, the same bits in each (one step for all
// numbers before the next: a result is not ready for another lane at once)
template <int NG, int N>
__device__ inline void ap4_over_groups(float (&x)[N]) {
    auto add = [&](auto ctrl) {
#pragma unroll
        for (int i = 0; i < N; i++)
            x[i] += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x[i]), decltype(ctrl)::value, 0xf, 0xf, true));
    };
    if constexpr (NG >= 2) add(std::integral_constant<int, 0x128>());  // 8 columns on
    if constexpr (NG >= 4) add(std::integral_constant<int, 0x124>());  // 4
    if constexpr (NG >= 8) add(std::integral_constant<int, 0x122>());  // 2
}

// The same for so few rows that the 16 columns of a tile can be NG groups of 32 dims times RB =
// 16 / NG rows: column group * RB + row. A column's query values are those of its group alone, so that
// a tile's score is the group's part of it, and a part is multiplied by the group's sub of its
// token where the key's scale is, in f32; the parts of a row are then added over its columns. The
// sums of values likewise: weights times subs are a column's operand, and of its sums the dims of its
// group are used. No code is multiplied by a sub: the subs of a token and its group are two numbers of a
// lane where the other kernel has eight, and their products with codes.
//
// Bound by memory and vector instructions at once: of a chunk's 640 instructions 290 make codes f16, the others are
// scores, weights and splits, of which NG columns have the same (vector pipes busy for two thirds of the time,
// matrix ones a fifth). 64 single tokens over up to 8192 keys, 32 heads of 128 on 8, 65 us in a loop (224 MB, 3.4 TB/s), 70 by
// the kernel above; one over 131072 41 (147 MB, 3.6 TB/s) and 44; 16 over up to 16000, 16 heads of 256 on 8, 77 and 92; 64 over
// up to 8192, 32 heads of 96, 56 and 61. Which of both runs is a matter of the columns: more rows do not fit (5 to 8 heads of
// 128 on each of 8 take 70 to 72 with the kernel above).
template <int KD, int NK, int ND, int TT, int WAVES, int NG>
__global__ __launch_bounds__(WAVES * 64, 2) void attnp4_groups_kernel(Attn4Args A) {
    constexpr int CH = 16 * TT, SEG = 4 * TT, KW = KD / 8, VW = SEG / 8, RB = 16 / NG;
    constexpr uint32_t kAll = (1u << SEG) - 1;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4, group = col / RB;
    const int hd = A.C.hd, shift = A.C.shift, B = 1 << shift;
    int r, h, tile, split, per;
    int64_t piece;
    Span s;
    if (!ap_rows_place(A, r, h, tile, split, per, piece, s)) return;
    const int32_t *table = A.R.table + (int64_t)r * A.R.max_blocks;
    const int n_tok = min(s.n, A.R.max_q), n_rows = n_tok * A.G;
    if (tile > 0 || n_rows <= 0) return;  // (the host launches it for up to RB rows)
    const Sight S = ap_sight(A, r, s, 0, n_tok - 1);
    const int n_split = ap_splits(A, S.n, per);
    if (split >= n_split) return;
    const int u0 = __builtin_amdgcn_readfirstlane((int)((int64_t)S.n * split / n_split));
    const int u1 = __builtin_amdgcn_readfirstlane((int)((int64_t)S.n * (split + 1) / n_split));
    auto chunk_of = [&](int u) { return ap4_chunk(S, u0, u1, u); };

    // table entries of this lane's key rows, and of its values and scores: loaded a chunk ahead,
    // between its keys and its values, and looked at when they are used (a wait for a load is one for
    // all loads before it)
    const int last_block = max(S.keys - 1, 0) >> shift, n_pages = (int)A.C.n_pages;
    auto first_of = [&](int u, int seg) { return chunk_of(u) * CH + seg * SEG; };
    auto entry_of = [&](int u, int seg) { return table[min(first_of(u, seg) >> shift, last_block)]; };
    auto page_of = [&](int u, int seg, int entry) { return first_of(u, seg) < S.keys && entry >= 0 && entry < n_pages ? entry : -1; };
    int u = u0 + wave, ek = 0, ev = 0, pv = 0;
    if (u < u1) {
        ek = entry_of(u, col >> 2);
        ev = entry_of(u, g);
    }

    // this lane's row
    const int row = min(col % RB, n_rows - 1);
    const int tok = row / A.G, head = h * A.G + row % A.G;
    const int p = s.p0 + tok;
    const float slope = A.slopes ? A.slopes[head] * kLog2e : 0.0f;
    const float *qrow = A.q + (s.q0 + tok) * A.ldq + (int64_t)head * hd;
    // this lane's dims of a key row; those past hd meet zeros of q
    auto dim_of = [&](int e) { return 4 * KD * e + KD * g; };
    float x[NK][KW][8];
#pragma unroll
    for (int e = 0; e < NK; e++)
#pragma unroll
        for (int y = 0; y < KW; y++) ap_load8(qrow + (dim_of(e) < hd ? dim_of(e) : 0) + 8 * y, A.q_vec, x[e][y]);

    // a chunk starts at a multiple of its length: a lane's place in a page is
    // its own and, in longer pages, the chunk's
    const int groups = hd / 32, kt = TT * col & (B - 1), vt = SEG * g & (B - 1);
    const uint32_t row_bytes = hd / 2, head_bytes = row_bytes << shift;
    const uint8_t *kb = (const uint8_t *)A.C.k + kt * row_bytes, *vb = (const uint8_t *)A.C.v + ((col << shift) + vt) / 2;
    uint32_t kr[TT][NK][KW], vr[ND][VW];
    uint32_t ksub[SEG / 4], vsub[SEG / 4], kd[SEG / 2], vd[SEG / 2];  // of this lane's tokens, subs of its group
    auto load_subs = [&](const int8_t *subs, int64_t ph, int at, uint32_t (&to)[SEG / 4]) {
        const int8_t *from = subs + ((ph * groups + min(group, groups - 1)) << shift) + at + vt;
        if constexpr (SEG == 16) {
            const ap_u4 v = *(const ap_u4 *)from;
#pragma unroll
            for (int e = 0; e < 4; e++) to[e] = v[e];
        } else {
            const uint2 v = *(const uint2 *)from;
            to[0] = v.x, to[1] = v.y;
        }
    };
    auto load_keys = [&](int u) {
        const int at = chunk_of(u) * CH & (B - 1), pk = page_of(u, col >> 2, ek);
        pv = page_of(u, g, ev);
        const int64_t ph = (int64_t)max(pk, 0) * A.C.n_kv + h, ps = (int64_t)max(pv, 0) * A.C.n_kv + h;
        const uint8_t *kp = kb + (ph * head_bytes + at * row_bytes);
#pragma unroll
        for (int e = 0; e < NK; e++) {
            const int d = dim_of(e) < hd ? dim_of(e) : 0;
#pragma unroll
            for (int t = 0; t < TT; t++) {
                if constexpr (KW == 4) {
                    const uint4 v = *(const uint4 *)(kp + t * row_bytes + d / 2);
                    kr[t][e][0] = v.x, kr[t][e][1] = v.y, kr[t][e][2] = v.z, kr[t][e][3] = v.w;
                } else {
                    const uint2 v = *(const uint2 *)(kp + t * row_bytes + d / 2);
                    kr[t][e][0] = v.x, kr[t][e][1] = v.y;
                }
            }
        }
        load_subs(A.ksub, ps, at, ksub);
        const ap_u4 *dk = (const ap_u4 *)(A.kd + (ps << shift) + at + vt), *dv = (const ap_u4 *)(A.vd + (ps << shift) + at + vt);
#pragma unroll
        for (int i = 0; i < SEG / 8; i++) {
            const ap_u4 a = dk[i], b = dv[i];
#pragma unroll
            for (int e = 0; e < 4; e++) kd[4 * i + e] = a[e], vd[4 * i + e] = b[e];
        }
    };
    auto load_values = [&](int u) {
        const int at = chunk_of(u) * CH & (B - 1);
        const int64_t ph = (int64_t)max(pv, 0) * A.C.n_kv + h;
        const uint8_t *vp = vb + (ph * head_bytes + at / 2);
#pragma unroll
        for (int d = 0; d < ND; d++) {
            const uint8_t *to = vp + (min(16 * d, hd - 16) << shift >> 1);
            if constexpr (VW == 2) {
                const uint2 v = *(const uint2 *)to;
                vr[d][0] = v.x, vr[d][1] = v.y;
            } else {
                vr[d][0] = *(const uint32_t *)to;
            }
        }
        load_subs(A.vsub, ph, at, vsub);
    };
    auto load_entries = [&](int u) {
        ek = entry_of(u, col >> 2);
        ev = entry_of(u, g);
    };
    if (u < u1) {
        load_keys(u);
        load_entries(min(u + WAVES, u1 - 1));
        load_values(u);
    }

    // the query, while the first keys are on their way
    ap_h8 qh[NK][KW], ql[NK][KW];
    float f_row, fc_row, turn;
    {
        // (no scale: zeros, so that a score is zero whatever the key)
        const float sign = A.scale2 > 0.0f ? A.sign : 0.0f;
        float amax = 0.0f;
#pragma unroll
        for (int e = 0; e < NK; e++)
#pragma unroll
            for (int y = 0; y < KW; y++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    x[e][y][j] = dim_of(e) < hd ? x[e][y][j] * sign : 0.0f;
                    amax = fmaxf(amax, fabsf(x[e][y][j]));
                }
        const int e2 = ap_row_exponent(ap_max_quarters(amax));
#pragma unroll
        for (int e = 0; e < NK; e++)
#pragma unroll
            for (int y = 0; y < KW; y++) {
#pragma unroll
                for (int j = 0; j < 8; j++) x[e][y][j] = dim_of(e) / 32 == group ? ldexpf(x[e][y][j], e2) : 0.0f;
                ap_split8(x[e][y], qh[e][y], ql[e][y]);
            }
        turn = ap4_factors(A, kAp4CodeBits - e2, -60, f_row, fc_row);
    }
    const bool turned = __any(turn != 1.0f);
    Running R;
    ap_f4 o[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) o[d] = ap_f4{0, 0, 0, 0};
    for (; u < u1; u += WAVES) {
        const int next = min(u + WAVES, u1 - 1), c = chunk_of(u);
        ap_f4 sc[TT];
#pragma unroll
        for (int t = 0; t < TT; t++) sc[t] = ap_f4{0, 0, 0, 0};
        // (two tiles at a time: a product waits for the one before it of its sum)
#pragma unroll
        for (int e = 0; e < NK; e++)
#pragma unroll
            for (int t = 0; t < TT; t += 2)
#pragma unroll
                for (int y = 0; y < KW; y++) {
                    ap_h8 a[2];
#pragma unroll
                    for (int i = 0; i < 2; i++) a[i] = ap4_codes(kr[t + i][e][y]);
#pragma unroll
                    for (int i = 0; i < 2; i++) sc[t + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[i], qh[e][y], sc[t + i], 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 2; i++) sc[t + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[i], ql[e][y], sc[t + i], 0, 0, 0);
                }
        if (turned) {
#pragma unroll
            for (int t = 0; t < TT; t++) sc[t] *= turn;
        }
        // key i of this lane: j0 + i; its score in log2 units is w[i] * f
        const int j0 = c * CH + g * SEG;
        float w[SEG], vs[SEG], f = f_row;
#pragma unroll
        for (int i = 0; i < SEG; i++) {
            w[i] = sc[i % TT][i / TT] * (ap4_bf16(kd[i / 2], i & 1) * ap4_byte(ksub[i / 4], i & 3));
            vs[i] = ap4_bf16(vd[i / 2], i & 1) * ap4_byte(vsub[i / 4], i & 3);
        }
        ap4_over_groups<NG>(w);
        const bool here = pv >= 0;
        load_keys(next);
        load_entries(min(next + WAVES, u1 - 1));
        if (A.cap != 0.0f) {
#pragma unroll
            for (int i = 0; i < SEG; i++) w[i] = ap_capped(A, w[i] * f, w[i] * fc_row);
            f = 1.0f;
        }
        if (A.slopes) {
            const float far = (float)(j0 - p);
#pragma unroll
            for (int i = 0; i < SEG; i++) w[i] = fmaf(w[i], f, -slope * fabsf(far + (float)i));
            f = 1.0f;
        }
        if (!ap_whole(A, S, c * CH, CH) || __any(!here)) {
            // (what was never written may have any scale)
            const uint32_t hidden = here ? ap_hidden(A, S, p, j0) & kAll : kAll;
#pragma unroll
            for (int i = 0; i < SEG; i++) {
                w[i] = ap_hide(w[i], hidden, i);
                vs[i] = hidden >> i & 1 ? 0.0f : vs[i];
            }
        }
        float mx = w[0];
#pragma unroll
        for (int i = 1; i < SEG; i++) mx = fmaxf(mx, w[i]);
        mx *= f;
        if (__any(mx > R.m + kApLate)) {
            const float ao = R.refer(R.raise(ap_max_quarters(mx)), 0.0f);
#pragma unroll
            for (int d = 0; d < ND; d++) o[d] *= ao;
        }
        // weights, and their products with the values' scales
        float z[SEG], most = 0.0f, few = 0.0f;
#pragma unroll
        for (int i = 0; i < SEG; i++) {
            const float x = __builtin_amdgcn_exp2f(fmaf(w[i], f, -R.m));
            few += x;
            z[i] = x * vs[i];
            most = fmaxf(most, fabsf(z[i]));
        }
        R.l += few;
        if (__any(most > 16.0f * R.ref)) {
            const float ao = R.refer(1.0f, ap_max_quarters(most));
#pragma unroll
            for (int d = 0; d < ND; d++) o[d] *= ao;
        }
        ap_h8 ph[VW], pl[VW];
#pragma unroll
        for (int e = 0; e < VW; e++) ap_split8w(z + 8 * e, R.over, ph[e], pl[e]);
#pragma unroll
        for (int d = 0; d < ND; d += 2)
#pragma unroll
            for (int e = 0; e < VW; e++) {
                const ap_h8 a = ap4_codes(vr[d][e]), b = ap4_codes(vr[d + 1][e]);
                o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ph[e], o[d], 0, 0, 0);
                o[d + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b, ph[e], o[d + 1], 0, 0, 0);
                o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pl[e], o[d], 0, 0, 0);
                o[d + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b, pl[e], o[d + 1], 0, 0, 0);
            }
        load_values(next);
    }
    ap_rows_end<ND, WAVES, RB>(A, s, R, o, kAp4Code / kApUnit, h, tile, n_rows, piece, split, n_split, tok, head);
}

// ---- many rows ---------------------------------------------------------------------
//
// attnp_tiles_kernel (attnp.h) over 4-bit values: the codes of a 64-key chunk become f16 numbers
// once, code * sub, on their way into LDS; the scales of its keys and values lie there beside
// them, as f32. A unit of 16 values is 8 bytes here.
//
// A wave has 32 rows. The scores of half a chunk are computed beside the weights of the half before, the products with
// values follow; two barriers a chunk. The queries' lower halves are read from LDS for each half: in
// registers they would leave none for the next scores.
//
// Bound by the vector step: vector instructions take 50% of the cycles (exponentials, four times as long, counted once) and
// products 42%, and a wave overlaps little of its own (two waves a SIMD are all that the registers allow). 3 prompts of up to 4096
// tokens behind up to 1000, 40 heads of 128 on 8, slopes and prefixes, 660-690 us: 425-445 TFLOP/s, twice that with the second
// halves, against the 1177 of a large f16 product; 4096 rows of 32 heads of 128 320-330, of 64 212-220. Four waves a block for
// heads up to 64 (with eight 252), eight for wider ones (with four, of whose blocks LDS holds one, 497). Waves without rows,
// chunks that a wave's rows do not see and what follows the last chunk take their turn with the others: nothing is skipped.
constexpr int ap4_tile_waves(int hd) { return hd <= 64 ? 4 : 8; }

template <int NS, int WAVES = ap4_tile_waves(16 * NS)>
__global__ __launch_bounds__(64 * WAVES, NS == 4 ? 3 : 2) void attnp4_tiles_kernel(Attn4Args A) {
    constexpr int kApTileRows = 32 * WAVES, kApTileThreads = 64 * WAVES;
    constexpr int ND = (NS + 1) / 2;             // 32-dim tiles of the output
    constexpr int KC = (2 * NS + 7) / 8 * 8;     // granules of a key row in LDS
    constexpr int NU = (64 * NS + kApTileThreads - 1) / kApTileThreads;  // 8-byte loads of a chunk, each
    __shared__ uint4 k_lds[2][64][KC];
    __shared__ uint4 v_lds[2][ND * 32][8];
    __shared__ uint4 q_lds[WAVES][NS][64];  // the lower halves of each wave's queries
    // scales of keys, times 2^-12, and values: a sum of 256 products of 2^14 and 1016 2^-16 times 2^116, the largest scale, is then a
    // number, and of the smallest one, 2^-110, no bits are lost
    __shared__ __attribute__((aligned(16))) float s_lds[2][2][64];
    constexpr int kScaleBits = 12;
    constexpr float kScaleUnit = 1.0f / (1 << kScaleBits);
    __shared__ __attribute__((aligned(16))) float m_lds[2][4];  // the largest scale of a segment of 16 values, -1 without a page
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, col = lane & 31, half = lane >> 5;
    const int hd = A.C.hd, shift = A.C.shift, B = 1 << shift;
    const int h = blockIdx.x % A.C.n_kv, split = blockIdx.y;
    const int64_t place = blockIdx.x / A.C.n_kv;
    int r = blockIdx.z, tile = (int)(A.n_tiles - 1 - place);
    if (A.placed && !ap_place(A, kApTileRows, place, r, tile)) return;
    const int64_t item = (A.placed ? place : (int64_t)r * A.n_tiles + tile) * A.C.n_kv + h;
    const Span s = request_span(A.R, r);
    const int n_tok = min(s.n, A.R.max_q), n_rows = n_tok * A.G;
    if (tile * kApTileRows >= n_rows) return;
    const Sight S = ap_sight(A, r, s, tile * kApTileRows / A.G, min((tile * kApTileRows + kApTileRows - 1) / A.G, n_tok - 1));
    const int n_split = ap_splits(A, S.n, A.per_split);
    if (split >= n_split) return;
    const int u0 = __builtin_amdgcn_readfirstlane((int)((int64_t)S.n * split / n_split));
    const int u1 = __builtin_amdgcn_readfirstlane((int)((int64_t)S.n * (split + 1) / n_split));
    auto chunk_of = [&](int u) { return ap4_chunk(S, u0, u1, u); };

    // the wave's rows and this lane's
    const int row0 = tile * kApTileRows + wave * 32;
    const int row = min(row0 + col, n_rows - 1), tok = row / A.G, head = h * A.G + row % A.G, p = s.p0 + tok;
    Sight W = S;
    W.p_lo = s.p0 + min(row0, n_rows - 1) / A.G;
    W.p_hi = s.p0 + min(row0 + 31, n_rows - 1) / A.G;
    const float slope = A.slopes ? A.slopes[head] * kLog2e : 0.0f;
    const float *qrow = A.q + (s.q0 + tok) * A.ldq + (int64_t)head * hd + 8 * half;

    // loads without branches: what is not there is read from elsewhere in the
    // table or the page and replaced
    const int32_t *table = A.R.table + (int64_t)r * A.R.max_blocks;
    const int last_block = max(S.keys - 1, 0) >> shift, n_pages = (int)A.C.n_pages;
    // (table entries are looked at when they are used: a wait for one is one for all loads before it)
    auto entry_of = [&](int j) { return table[min(j >> shift, last_block)]; };
    auto page_of = [&](int j, int entry) { return j < S.keys && entry >= 0 && entry < n_pages ? entry : -1; };
    // this thread's parts of a chunk: 16 dims of a key, and eight keys of two dims (which share
    // their subs); a scale, of threads 0 .. 63 a key's, 64 .. 127 a value's
    constexpr bool kWhole = 64 * NS % kApTileThreads == 0;
    auto unit = [&](int i) { return kWhole ? tid + kApTileThreads * i : min(tid + kApTileThreads * i, 64 * NS - 1); };
    const int n_kv = A.C.n_kv, seg = 16 * (tid >> 1 & 3), scaled = seg + (tid >> 2 & 14) + (tid & 1);
    const uint32_t row_bytes = hd / 2, head_bytes = row_bytes << shift, page_bytes = head_bytes * (uint32_t)n_kv;
    const uint32_t page_subs = page_bytes / 16, page_scales = (uint32_t)n_kv << shift;
    uint32_t koff[NU], ksoff[NU], voff[NU], vsoff[NU];  // in a page, without the chunk's place
    uint32_t kr[NU][2], ksub[NU], vr[NU][2], vsub[NU][2], scale;
    int ek[NU], ev, vpg = -1;  // entries; the page of this thread's values and scale
    bool seen = false;         // some row may see the key of `scale`
    const int seen_to = min(S.keys, max(S.p_hi + 1, S.prefix));
#pragma unroll
    for (int i = 0; i < NU; i++) {
        const int key = unit(i) / NS, d = unit(i) % NS * 16 < hd ? unit(i) % NS * 16 : 0;
        const int dim = unit(i) >> 3 << 1 < hd ? unit(i) >> 3 << 1 : 0, v0 = 8 * (tid & 7) & (B - 1);
        koff[i] = h * head_bytes + (key & (B - 1)) * row_bytes + d / 2;
        ksoff[i] = (uint32_t)((h * (hd / 32) + d / 32) << shift) + (key & (B - 1));
        voff[i] = h * head_bytes + ((dim << shift) + v0) / 2;
        vsoff[i] = (uint32_t)((h * (hd / 32) + dim / 32) << shift) + v0;
    }
    const uint32_t soff = (uint32_t)(h << shift) + (scaled & (B - 1));
    auto load_entries = [&](int u) {
        const int j0 = chunk_of(u) * 64;
#pragma unroll
        for (int i = 0; i < NU; i++) ek[i] = entry_of(j0 + unit(i) / NS);
        ev = entry_of(j0 + seg);
    };
    auto load_keys = [&](int u) {
        const int j0 = chunk_of(u) * 64, at = j0 & (B - 1);
#pragma unroll
        for (int i = 0; i < NU; i++) {
            const uint64_t pg = (uint32_t)max(page_of(j0 + unit(i) / NS, ek[i]), 0);
            const uint2 v = *(const uint2 *)((const uint8_t *)A.C.k + (pg * page_bytes + at * row_bytes + koff[i]));
            kr[i][0] = v.x, kr[i][1] = v.y;
            ksub[i] = *(const uint8_t *)(A.ksub + (pg * page_subs + at + ksoff[i]));
        }
        vpg = page_of(j0 + seg, ev);
        // (what no row sees may have any scale, and counts as zero: also new tokens behind the block's last row, which
        // nothing has written where they are past max_q)
        const int j = j0 + scaled;
        seen = vpg >= 0 && j < seen_to && (!A.window || j > S.p_lo - A.window || j < S.prefix);
        if (tid < 128) scale = (tid < 64 ? A.kd : A.vd)[(uint64_t)(uint32_t)max(vpg, 0) * page_scales + at + soff];
    };
    auto load_values = [&](int u) {
        const int at = chunk_of(u) * 64 & (B - 1);
        const uint64_t pg = (uint32_t)max(vpg, 0);
#pragma unroll
        for (int i = 0; i < NU; i++) {
            const uint8_t *from = (const uint8_t *)A.C.v + (pg * page_bytes + at / 2 + voff[i]);
            vr[i][0] = *(const uint32_t *)from;
            vr[i][1] = *(const uint32_t *)(from + (B >> 1));
            const uint2 v = *(const uint2 *)(A.vsub + (pg * page_subs + at + vsoff[i]));
            vsub[i][0] = v.x, vsub[i][1] = v.y;
        }
    };
    auto put_keys = [&](int buf) {
#pragma unroll
        for (int i = 0; i < NU; i++) {
            const int key = unit(i) / NS, d16 = unit(i) % NS;
            // (dims past hd meet zeros of q: they must be numbers, and any code and sub make one)
            Ap4Sub s[4];
            ap4_sub(ksub[i], 0, s);
            const int kx = (key & 3) | ((key >> 2) & 4) | ((key << 1) & 8), x = KC % 16 ? kx >> 1 : kx;
            k_lds[buf][key][(2 * d16) ^ x] = __builtin_bit_cast(uint4, ap4_cvt(kr[i][0], s));
            k_lds[buf][key][(2 * d16 + 1) ^ x] = __builtin_bit_cast(uint4, ap4_cvt(kr[i][1], s));
        }
        if (tid < 128) {
            const float x = seen ? ap4_bf16(scale, 0) : 0.0f;
            s_lds[buf][tid >> 6][scaled] = tid < 64 ? x * kScaleUnit : x;
            // the segment's 16 values are those of the lanes that differ in bits 0, 3, 4 and 5
            float most = fmaxf(x, kv4_from<0xb1>(x));
            most = fmaxf(most, kv4_from<0x128>(most));
            most = ap_max_quarters(most);
            if (tid >= 64 && tid < 72) m_lds[buf][tid >> 1 & 3] = vpg >= 0 ? most : -1.0f;
        }
    };
    auto put_values = [&](int buf) {
#pragma unroll
        for (int i = 0; i < NU; i++) {
            const int dim = unit(i) >> 3 << 1, y = (dim >> 1) & 7;
            Ap4Sub s[4];
            ap4_subs(vsub[i][0], vsub[i][1], s);
            v_lds[buf][dim][(tid & 7) ^ y] = __builtin_bit_cast(uint4, ap4_cvt(vr[i][0], s));
            v_lds[buf][dim + 1][(tid & 7) ^ y] = __builtin_bit_cast(uint4, ap4_cvt(vr[i][1], s));
        }
    };

    Running R;
    if (u0 < u1) {
        load_entries(u0);
        load_keys(u0);
        load_entries(min(u0 + 1, u1 - 1));
        load_values(u0);
    }
    // the query, while the first chunk is on its way
    ap_h8 qh[NS];
    float f_row, fc_row;
    {
        const float sign = A.scale2 > 0.0f ? A.sign : 0.0f;  // (no scale: a score is zero whatever the key)
        float x[NS][8], amax = 0.0f;
#pragma unroll
        for (int c = 0; c < NS; c++) ap_load8(qrow + (16 * c < hd ? 16 * c : 0), A.q_vec, x[c]);
#pragma unroll
        for (int c = 0; c < NS; c++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                x[c][j] = 16 * c < hd ? x[c][j] * sign : 0.0f;
                amax = fmaxf(amax, fabsf(x[c][j]));
            }
        const int e2 = ap_row_exponent(ap_max_halves(amax));
#pragma unroll
        for (int c = 0; c < NS; c++) {
#pragma unroll
            for (int j = 0; j < 8; j++) x[c][j] = ldexpf(x[c][j], e2);
            ap_h8 lo;
            ap_split8(x[c], qh[c], lo);
            q_lds[wave][c][lane] = __builtin_bit_cast(uint4, lo);
        }
        if (ap4_factors(A, kAp4Bits + kScaleBits - e2, INT_MIN, f_row, fc_row) != 1.0f) f_row = -f_row;
    }
    // (large rows have the sign of f_row, taken off for each half: a mask of their own, or one more branch, makes heads of 64 spill,
    // 4096 rows 225 us and not 214)
    const bool capped_or_large = __any(f_row < 0.0f) || A.cap != 0.0f;
    ap_f16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[d][i] = 0.0f;
    // where this lane's operands lie in LDS: the granules of a row are permuted by an exclusive or, so
    // that another granule is another exclusive or of the address. The empty statements keep
    // the compiler from holding all of these in registers, which the operands need.
    const int key = 16 * ((col >> 2) & 1) + 4 * (col >> 3) + (col & 3);
    const uint32_t k_at = key * KC * 16 + ((half ^ (KC % 16 ? (col >> 1) & 7 : col & 15)) << 4);
    const uint32_t v_at = col * 128 + ((2 * half ^ ((col >> 1) & 7)) << 4);
    auto scores = [&](ap_f16 &sc, int buf, int i) {
        uint32_t at = k_at + (64 * buf + 32 * i) * KC * 16;
        asm("" : "+v"(at));
#pragma unroll
        for (int e = 0; e < 16; e++) sc[e] = 0.0f;
#pragma unroll
        for (int c = 0; c < NS; c++) {
            const ap_h8 a = *(const ap_h8 *)((const char *)k_lds + (at ^ c << 5));
            sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qh[c], sc, 0, 0, 0);
            sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, __builtin_bit_cast(ap_h8, q_lds[wave][c][lane]), sc, 0, 0, 0);
        }
    };
    ap_f16 sc;
    if (u0 < u1) {
        put_keys(0);
        put_values(0);
        load_keys(min(u0 + 1, u1 - 1));
        load_entries(min(u0 + 2, u1 - 1));
        load_values(min(u0 + 1, u1 - 1));
        __syncthreads();
        scores(sc, 0, 0);
    }
    for (int u = u0; u < u1; u++) {
        const int buf = (u - u0) & 1, j0 = chunk_of(u) * 64;
        const bool whole = ap_whole(A, W, j0, 64);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            {
                // scores in log2 units are sc * f
                const float4 vm = *(const float4 *)m_lds[buf];
                const float vmax = i == 0 ? (half ? vm.y : vm.x) : (half ? vm.w : vm.z);
                const float *kd = &s_lds[buf][0][32 * i + 16 * half], *vd = &s_lds[buf][1][32 * i + 16 * half];
                float f = f_row;
                asm("" : "+v"(f));
                const bool large = f < 0.0f;
                f = fabsf(f);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float4 d = ((const float4 *)kd)[e];
                    sc[4 * e] *= d.x, sc[4 * e + 1] *= d.y, sc[4 * e + 2] *= d.z, sc[4 * e + 3] *= d.w;
                }
                if (capped_or_large) {
                    if (__any(large)) {
#pragma unroll
                        for (int e = 0; e < 16; e++) sc[e] = large ? sc[e] * 0x1p64f : sc[e];
                    }
                    if (A.cap != 0.0f) {
#pragma unroll
                        for (int e = 0; e < 16; e++) sc[e] = ap_capped(A, sc[e] * f, sc[e] * fc_row);
                        f = 1.0f;
                    }
                }
                const int j1 = j0 + 32 * i + 16 * half;
                if (A.slopes) {
                    const float far = (float)(j1 - p), base = slope * far;
                    if (j0 + 63 <= W.p_lo) {  // no key behind a row's own
#pragma unroll
                        for (int e = 0; e < 16; e++) sc[e] = fmaf(sc[e], f, fmaf(slope, (float)e, base));
                    } else {
#pragma unroll
                        for (int e = 0; e < 16; e++) sc[e] = fmaf(sc[e], f, -slope * fabsf(far + (float)e));
                    }
                    f = 1.0f;
                }
                if (!whole || __any(vmax < 0.0f)) {
                    const uint32_t hidden = vmax < 0.0f ? 0xffffu : ap_hidden(A, S, p, j1);
#pragma unroll
                    for (int e = 0; e < 16; e++) sc[e] = ap_hide(sc[e], hidden, e);
                }
                float mx = sc[0];
#pragma unroll
                for (int e = 1; e < 16; e++) mx = fmaxf(mx, sc[e]);
                mx *= f;
                // no product of a weight and its scale is more than the largest weight times the
                // largest scale: only where that passes the reference the products are looked at
                int late = __any(R.late(mx, __builtin_amdgcn_exp2f(fminf(mx - R.m, kApLate)) * vmax));
                while (late) {
                    const float am = R.raise(ap_max_halves(mx));
                    float most = 0.0f;
#pragma unroll
                    for (int e = 0; e < 16; e++) most = fmaxf(most, __builtin_amdgcn_exp2f(fmaf(sc[e], f, -R.m)) * vd[e]);
                    const float ao = R.refer(am, ap_max_halves(most));
#pragma unroll
                    for (int d = 0; d < ND; d++) o[d] *= ao;
                    late = 0;
                    asm("" : "+s"(late));
                }
                asm("" : "+v"(R.m));
                // the next half's scores (behind the last chunk: of what is there, for nobody) beside the weights
                ap_f16 next;
                scores(next, i == 0 ? buf : buf ^ 1, i ^ 1);
                // (16 weights are added first: a sum of thousands, one by one, is off by more than the products)
                float z[16], l16 = 0.0f;
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const float w = __builtin_amdgcn_exp2f(fmaf(sc[e], f, -R.m));
                    l16 += w;
                    z[e] = w * vd[e];
                }
                R.l += l16;
                ap_h8 ph[2], pl[2];
#pragma unroll
                for (int e = 0; e < 2; e++) ap_split8w(z + 8 * e, R.over, ph[e], pl[e]);
                // and their products with the values
                uint32_t at = v_at + buf * ND * 32 * 128;
                asm("" : "+v"(at));
#pragma unroll
                for (int e = 0; e < 2; e++)
#pragma unroll
                    for (int d = 0; d < ND; d++) {
                        const ap_h8 a = *(const ap_h8 *)((const char *)v_lds + ((at ^ (4 * i + e) << 4) + d * 4096));
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ph[e], o[d], 0, 0, 0);
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, pl[e], o[d], 0, 0, 0);
                    }
                sc = next;
            }
            if (i == 0) {
                put_keys(buf ^ 1);
                load_keys(min(u + 2, u1 - 1));
                load_entries(min(u + 3, u1 - 1));
            } else {
                put_values(buf ^ 1);
                load_values(min(u + 2, u1 - 1));
            }
            __syncthreads();
        }
    }
    float m, l = R.l;
    l += __shfl_xor(l, 32);

    const float back = ap_unit(R, kAp4Unit / kApUnit, m, l);
    if (row0 + col < n_rows) {
        // four dims in a row a register group: 32 d + 8 a + 4 half ..
        if (n_split == 1) {
            float *to = A.out + (s.q0 + tok) * A.ldo + (int64_t)head * hd + 4 * half;
            const float z = l > 0.0f || l != l ? back / l : 0.0f;
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int a = 0; a < 4; a++)
                    if (32 * d + 8 * a < hd) ap_put4(to + 32 * d + 8 * a, o[d][4 * a] * z, o[d][4 * a + 1] * z,
                                o[d][4 * a + 2] * z, o[d][4 * a + 3] * z, A.out_vec);
        } else {
            float4 *to = ap_part(A, item * A.n_split + split, kApTileRows) + wave * 32 + col;
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int a = 0; a < 4; a++)
                    if (32 * d + 8 * a < hd)
                        to[(8 * d + 2 * a + half) * kApTileRows] = float4{o[d][4 * a] * back, o[d][4 * a + 1] * back,
                                                                          o[d][4 * a + 2] * back, o[d][4 * a + 3] * back};
            if (half == 0) to[hd / 4 * kApTileRows] = float4{m, l, 0, 0};
        }
    }
}

}  // namespace sihip
