// Attention over the paged 4-bit KV cache (kvcache4.h): the mathematics, row blocks,
// pieces and running softmax of attnp.h, over values code * sub * scale.
//
// code * sub is a whole number up to 1016 in magnitude and exact in f16, so the matrix
// cores get it as one operand, and the f32 operand split into two f16 numbers as
// for the 8-bit cache: results are of f32 accuracy. A nibble n (a code plus 8), put at bits 6 to 9 of
// 0x4c00, is the f16 number 16 + n, and one packed FMA, (16 + n) sub - 24 sub, is
// (n - 8) sub without a rounding: three instructions for two values, where
// the bytes of the 8-bit cache take two and a half. What is left of a key's and a
// value's scale is one factor a token: scores are multiplied by the key's, weights by the
// value's before they are split.
#pragma once

#include "attnp.h"
#include "kvcache4.h"

namespace sihip {

// C: of the cache, with codes in place of bytes and no scales
struct Attn4Args : AttnPArgs {
    const int8_t *ksub, *vsub;
    const uint16_t *kd, *vd;
};

typedef uint32_t ap_u4 __attribute__((ext_vector_type(4)));

// eight nibbles times the subs of their elements: s[i] (and m[i] = -24 s[i]) of elements 2 i and 2 i + 1
__device__ inline ap_h8 ap4_cvt(uint32_t w, const ap_h2 (&s)[4], const ap_h2 (&m)[4]) {
    union {
        ap_h8 v;
        ap_h2 h[4];
    } u;
    const uint32_t n[4] = {w << 6, w << 2, w >> 2, w >> 6};
#pragma unroll
    for (int i = 0; i < 4; i++)
        u.h[i] = __builtin_elementwise_fma(__builtin_bit_cast(ap_h2, (n[i] & 0x03c003c0u) | 0x4c004c00u), s[i], m[i]);
    return u.v;
}

// byte t of x (a sub) as both halves of a pair, and -24 times it
__device__ inline void ap4_sub(uint32_t x, int t, ap_h2 &s, ap_h2 &m) {
    const ap_h2 off = {(_Float16)1152.0f, (_Float16)1152.0f}, f = {(_Float16)-24.0f, (_Float16)-24.0f};
    s = __builtin_bit_cast(ap_h2, __builtin_amdgcn_perm(0x64646464u, x ^ 0x80808080u, 0x04000400u | (uint32_t)t * 0x00010001u)) - off;
    m = s * f;
}

// a bfloat16 in the low or high half of x
__device__ inline float ap4_bf16(uint32_t x, int high) { return __builtin_bit_cast(float, high ? x & 0xffff0000u : x << 16); }

// ---- few rows ----------------------------------------------------------------------
//
// attnp_rows_kernel (attnp.h) over 4-bit values: 16 rows of one request and KV head, one split of
// its chunks of 16 TT keys, global memory to registers. KD dims of a key are a lane's in each of
// NK slices of 4 KD: 16 bytes, or 8 for heads up to 64. Row m of key tile t is token TT m + t, so
// that a lane's TT subs are neighbours, and its scores, of tokens 4 TT g .., are
// i-major: token TT i + t of them is register (t, i).
template <int KD, int NK, int ND, int TT, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 2) void attnp4_rows_kernel(Attn4Args A) {
    constexpr int CH = 16 * TT, SEG = 4 * TT, KW = KD / 8, VW = SEG / 8;
    constexpr uint32_t kAll = (1u << SEG) - 1;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
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
    const int u0 = (int)((int64_t)S.n * split / n_split), u1 = (int)((int64_t)S.n * (split + 1) / n_split);

    // pages of this lane's key rows, and of its values and scores
    const int last_block = max(S.keys - 1, 0) >> shift, n_pages = (int)A.C.n_pages;
    auto page_of = [&](int u, int seg) {
        const int j = ap_chunk(S, u) * CH + seg * SEG, pg = table[min(j >> shift, last_block)];
        return j < S.keys && pg >= 0 && pg < n_pages ? pg : -1;
    };
    int u = u0 + wave, pk = 0, pv = 0;
    if (u < u1) {
        pk = page_of(u, col >> 2);
        pv = page_of(u, g);
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
    bool some = false;  // this lane's segment has a page
    auto load_keys = [&](int u) {
        const int at = ap_chunk(S, u) * CH & (B - 1);
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
        some = pv >= 0;
    };
    auto load_values = [&](int u, int page) {
        const int at = ap_chunk(S, u) * CH & (B - 1);
        const int64_t ph = (int64_t)max(page, 0) * A.C.n_kv + h;
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
    if (u < u1) {
        load_keys(u);
        load_values(u, pv);
        const int next = min(u + WAVES, u1 - 1);
        pk = page_of(next, col >> 2);
        pv = page_of(next, g);
    }

    // the query, while the first keys are on their way
    ap_h8 qh[NK][KW], ql[NK][KW];
    float f_row, fc_row;
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
        f_row = ldexpf(1.0f, -e2);
        fc_row = fminf(f_row * A.cap_in, FLT_MAX);
        f_row = fmaxf(f_row * A.scale2, FLT_MIN);  // above zero: it leaves -inf as it is
    }
    Running R;
    ap_f4 o[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) o[d] = ap_f4{0, 0, 0, 0};
    for (; u < u1; u += WAVES) {
        const int next = min(u + WAVES, u1 - 1), c = ap_chunk(S, u);
        ap_f4 sc[TT];
#pragma unroll
        for (int t = 0; t < TT; t++) sc[t] = ap_f4{0, 0, 0, 0};
        // (two tiles at a time: a product waits for the one before it of its sum)
#pragma unroll
        for (int e = 0; e < NK; e++)
#pragma unroll
            for (int t = 0; t < TT; t += 2) {
                ap_h2 sub[2][4], m[2][4];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    ap4_sub(ksub[e], t + i, sub[i][0], m[i][0]);
#pragma unroll
                    for (int k = 1; k < 4; k++) sub[i][k] = sub[i][0], m[i][k] = m[i][0];
                }
#pragma unroll
                for (int y = 0; y < KW; y++) {
                    ap_h8 a[2];
#pragma unroll
                    for (int i = 0; i < 2; i++) a[i] = ap4_cvt(kr[t + i][e][y], sub[i], m[i]);
#pragma unroll
                    for (int i = 0; i < 2; i++) sc[t + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[i], qh[e][y], sc[t + i], 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 2; i++) sc[t + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[i], ql[e][y], sc[t + i], 0, 0, 0);
                }
            }
        // key i of this lane: j0 + i; its score in log2 units is w[i] * f
        const int j0 = c * CH + g * SEG;
        float w[SEG], vs[SEG], f = f_row;
#pragma unroll
        for (int i = 0; i < SEG; i++) {
            w[i] = sc[i % TT][i / TT] * ap4_bf16(kd[i / 2], i & 1);
            vs[i] = ap4_bf16(vd[i / 2], i & 1);
        }
        const bool here = some;
        const int pv_next = pv;
        load_keys(next);
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
        // weights, and their products with the values' scales
        float pr[SEG], z[SEG], most = 0.0f;
#pragma unroll
        for (int i = 0; i < SEG; i++) {
            pr[i] = __builtin_amdgcn_exp2f(fmaf(w[i], f, -R.m));
            z[i] = pr[i] * vs[i];
            most = fmaxf(most, z[i]);
        }
        if (__any(R.late(mx, most))) {
            const float am = R.raise(ap_max_quarters(mx));
            most = 0.0f;
#pragma unroll
            for (int i = 0; i < SEG; i++) {
                pr[i] = __builtin_amdgcn_exp2f(fmaf(w[i], f, -R.m));
                z[i] = pr[i] * vs[i];
                most = fmaxf(most, z[i]);
            }
            const float ao = R.refer(am, ap_max_quarters(most));
#pragma unroll
            for (int d = 0; d < ND; d++) o[d] *= ao;
        }
        ap_h8 ph[VW], pl[VW];
#pragma unroll
        for (int e = 0; e < VW; e++) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                R.l += pr[8 * e + j];
                z[8 * e + j] *= R.over;  // a power of two
            }
            ap_split8(z + 8 * e, ph[e], pl[e]);
        }
#pragma unroll
        for (int d = 0; d < ND; d += 2) {
            ap_h2 sub[VW][4], m[VW][4];
#pragma unroll
            for (int e = 0; e < VW; e++) {
                const ap_h2 k24 = {(_Float16)-24.0f, (_Float16)-24.0f};
                ap_cvt4(vsub[d / 2][2 * e], sub[e][0], sub[e][1]);
                ap_cvt4(vsub[d / 2][2 * e + 1], sub[e][2], sub[e][3]);
#pragma unroll
                for (int k = 0; k < 4; k++) m[e][k] = sub[e][k] * k24;
            }
#pragma unroll
            for (int e = 0; e < VW; e++) {
                const ap_h8 a = ap4_cvt(vr[d][e], sub[e], m[e]), b = ap4_cvt(vr[d + 1][e], sub[e], m[e]);
                o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ph[e], o[d], 0, 0, 0);
                o[d + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b, ph[e], o[d + 1], 0, 0, 0);
                o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pl[e], o[d], 0, 0, 0);
                o[d + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b, pl[e], o[d + 1], 0, 0, 0);
            }
        }
        load_values(next, pv_next);
        pk = page_of(min(next + WAVES, u1 - 1), col >> 2);
        pv = page_of(min(next + WAVES, u1 - 1), g);
    }
    ap_rows_end<ND, WAVES>(A, s, R, o, h, tile, n_rows, piece, split, n_split, tok, head);
}

}  // namespace sihip
