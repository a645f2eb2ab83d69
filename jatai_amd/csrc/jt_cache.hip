// The paged key-value cache of generation (no reference counterpart: the reference only trains): its page operators, and
// attention of new tokens over it.
//
// The cache is a block tensor laid out in pages: m int8 [pages][layers][2: keys, values][Hk][pag][hd] and E int8 [pages]
// [layers][2][Hk][pag][G], G = hd / GS exponents per token and head, GS = min(hd, BLK) values each. A (page, head) is one
// contiguous tile of pag x hd bytes. pag is a power of two from 16 on; a token at position j of sequence b is slot j % pag
// of page tab[b][j / pag]. The bytes are those of the model's Q/K/V product, copied, so nothing is rounded on the way in.
//
// Rows of a call: sequence b has the rows ini[b] .. ini[b + 1] - 1 of a block tensor [M, (H + 2 Hk) hd] (q, k, v side by
// side), which are its newest tokens, at positions comp[b] - (ini[b + 1] - ini[b]) .. comp[b] - 1. Lengths and tables are
// read on the device, so a captured graph follows them. What they say is checked there: a malformed sequence or a page
// outside the cache raises E_ARG, reads nothing and counts as not visible.
#include "jt_comum.h"

namespace atc {
struct Seq { int b, i, ok; };                    // sequence of a row, its position, whether it has one

struct Lote {
    const int *tab, *comp, *ini;                 // [B][P], [B], [B + 1]; ini null: row b is sequence b's
    int B, P, M, lgpag, npag, novos, teto;       // novos: most rows of a sequence; teto: most tokens
};

// first row, row count and length of sequence b; false where they are malformed
__device__ __forceinline__ bool sequencia(const Lote& L, int b, int& r0, int& n, int& comp) {
    comp = L.comp[b];
    r0 = L.ini ? L.ini[b] : b;
    n = L.ini ? L.ini[b + 1] - r0 : min(comp, 1);                     // without starts, an empty sequence has no row
    return r0 >= 0 && n >= 0 && r0 <= L.M - n && n <= L.novos && comp >= n && comp <= L.teto;
}

// E_ARG for every malformed sequence, by one workgroup of a launch: a sequence that nobody comes upon by a row of its own (starts that
// fall back) is found here
__device__ __forceinline__ void confere(const Lote& L, int kid, int parte, int passo) {
    int r0, n, comp;
    for (int b = parte; b < L.B; b += passo)
        if (!sequencia(L, b, r0, n, comp)) reporta(E_ARG, kid, r0, comp, b);
}

// The sequence of row r, found by a whole wave: every lane looks at one of 64 starts, and the last start at or below r
// is counted. One memory round trip, where a binary search takes one per step.
__device__ __forceinline__ int sequencia_de(const Lote& L, int r) {
    if (!L.ini) return r < L.B ? r : -1;
    int n = 0;
    for (int k = 0; k < L.B; k += 64) {
        const int x = k + (int)(threadIdx.x & 63);
        n += __popcll(__ballot(x < L.B && L.ini[min(x, L.B)] <= r));
    }
    return n - 1 >= 0 && r < L.ini[n] ? n - 1 : -1;
}

// the same with the sequence's own numbers, which the lanes load beside the starts: still one round trip
__device__ __forceinline__ Seq acha(const Lote& L, int r) {
    Seq s{-1, 0, 0};
    int r0 = r, fim = r + 1, comp = 0;
    if (L.ini) {
        for (int k = 0; k < L.B; k += 64) {
            const int x = k + (int)(threadIdx.x & 63), a = L.ini[min(x, L.B)], b = L.ini[min(x + 1, L.B)], c = L.comp[min(x, L.B - 1)];
            const int n = __popcll(__ballot(x < L.B && a <= r));
            if (n == 0) break;
            s.b = k + n - 1;
            r0 = __shfl(a, n - 1);
            fim = __shfl(b, n - 1);
            comp = __shfl(c, n - 1);
            if (n < 64) break;
        }
        if (r >= fim) s.b = -1;
    } else if (r < L.B) {
        s.b = r;
        comp = L.comp[r];
        fim = r + min(comp, 1);                                       // an empty sequence has no row
    }
    if (s.b < 0) return s;
    const int n = fim - r0;
    s.ok = r0 >= 0 && n >= 0 && r0 <= L.M - n && n <= L.novos && comp >= n && comp <= L.teto;
    s.ok = s.ok && r - r0 < n;
    s.i = comp - n + (r - r0);
    return s;
}
}  // namespace atc

// ---------------------------------------------------------------------------------------------- pages
// The rows' keys and values into their slots. A thread moves VB bytes (a head's 16, or its 4): the threads of a wave hold
// the same chunks of consecutive rows, whose slots are consecutive, so a wave writes whole kilobytes of a page's tile.
// Bound by its bytes, read and written once: 16 prompts of 300 to 2048 tokens, 8 heads of 64, 10.9 us (3.7 TB/s, the launch's start and
// end included); 32 rows 3.7 us, the launch and two reads that wait for each other.
template <int HD, int GS>
__global__ void __launch_bounds__(256) k_cache_grava(const int8_t* __restrict__ qm, const int8_t* __restrict__ qE, int8_t* __restrict__ cm,
                                                     int8_t* __restrict__ cE, atc::Lote L, int H, int Hk, int lgblk, long long pag_m,
                                                     long long pag_e, int kid) {
    constexpr int VB = HD < 16 ? HD : 16, NC = HD / VB, G = HD / GS, LPW = 64 / NC;     // LPW: rows per wave
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int r = blockIdx.x * LPW + lane / NC, c = lane % NC;
    const int kvh = blockIdx.y * 4 + w;                                                 // keys' heads, then values'
    if (blockIdx.x == gridDim.x - 1) {                                                  // has no rows
        if (blockIdx.y == 0) atc::confere(L, kid, threadIdx.x, 256);
        return;
    }
    if (kvh >= 2 * Hk) return;
    // one search per wave for its first row; the rows after it follow
    int b = atc::sequencia_de(L, min((int)(blockIdx.x * LPW), L.M - 1));
    if (r >= L.M) return;
    if (L.ini) {
        if (b < 0) b = 0;
        while (b < L.B && r >= L.ini[b + 1]) b++;
        if (b >= L.B || r < L.ini[b]) return;                                           // behind the last sequence
    } else if ((b = r) >= L.B) return;
    int r0, n, comp;
    if (!atc::sequencia(L, b, r0, n, comp) || r - r0 >= n) return;
    const int j = comp - n + (r - r0), pag = 1 << L.lgpag;
    const int p = L.tab[(long long)b * L.P + (j >> L.lgpag)];
    if ((unsigned)p >= (unsigned)L.npag) {
        if (kvh == 0 && c == 0) reporta(E_ARG, kid, (long long)b * L.P + (j >> L.lgpag), p, j);
        return;
    }
    const int ld = (H + 2 * Hk) * HD, col = (H + kvh) * HD + c * VB;
    const long long vaga = (long long)kvh * pag + (j & (pag - 1));
    const int8_t* de = qm + (long long)r * ld + col;
    int8_t* para = cm + p * pag_m + vaga * HD + c * VB;
    if constexpr (VB == 16) *reinterpret_cast<int4*>(para) = *reinterpret_cast<const int4*>(de);
    else *reinterpret_cast<int*>(para) = *reinterpret_cast<const int*>(de);
    if (c * VB % GS == 0) cE[p * pag_e + vaga * G + c * VB / GS] = qE[(long long)r * (ld >> lgblk) + (col >> lgblk)];
}

// Whole pages copied, up to PARES_COPIA pairs by value in the launch's arguments (nothing to upload, and a captured graph
// keeps them). The pairs' targets are distinct and no pair's source, which the host has checked. Bound by its bytes: 300 pages
// of 12 layers (811 KB each) 92 us, 5.3 TB/s, what a large copy reaches.
constexpr int PARES_COPIA = 256;
struct ParesCopia { int de[PARES_COPIA], para[PARES_COPIA]; };
__global__ void __launch_bounds__(256) k_cache_copia(int8_t* __restrict__ cm, int8_t* __restrict__ cE, ParesCopia ps, long long pag_m, long long pag_e) {
    const long long d = ps.de[blockIdx.y], p = ps.para[blockIdx.y];
    const int4 *dm = reinterpret_cast<const int4*>(cm + d * pag_m), *de = reinterpret_cast<const int4*>(cE + d * pag_e);
    int4 *pm = reinterpret_cast<int4*>(cm + p * pag_m), *pe = reinterpret_cast<int4*>(cE + p * pag_e);
    const long long nm = pag_m / 16, ne = pag_e / 16;
    for (long long k = (long long)blockIdx.x * 256 + threadIdx.x; k < nm + ne; k += (long long)gridDim.x * 256)
        if (k < nm) pm[k] = dm[k];
        else pe[k - nm] = de[k - nm];
}

// ---------------------------------------------------------------------------------------------- attention
namespace atc {
struct Args {
    const int8_t *qm, *qE, *cm, *cE;             // cm, cE: at the layer
    const float* incl;                           // null: no bias
    float *ml, *o;                               // partial results: (maximum, sum) and outputs per (row, head, split); null:
    void* out;                                   // none, the kernel itself writes out (outE) as `tipo` (k_atc_junta's) says
    int8_t* outE;
    long long pag_m, pag_e;
    Lote L;
    bool inteira;                                // the blocks of a block output lie in one head each
    int H, Hk, lgblk, janela, sumid, S, fatia, tipo, kid;   // S splits of `fatia` tiles of visible tokens each
};

// a page outside the cache that the token at position `ruim` (-1: none) of sequence b needed
__device__ __forceinline__ void relata_pagina(const Args& a, int b, int ruim) {
    if (ruim < 0) return;
    const long long x = (long long)b * a.L.P + (ruim >> a.L.lgpag);
    reporta(E_ARG, a.kid, x, a.L.tab[x], ruim);
}

// Scores stay in nats (a factor of log2 e would round each of them once more) and become powers of two as
// exp2(s log2 e - m log2 e), one FMA whose rounding is small where the weight is large. The rounding of m log2 e is common to
// all weights under a maximum, and the factor between two maxima takes the same rounded products (never contracted into an FMA), so that
// it fits them, and is exactly 1 where the maximum stays.
// k_atc_mf keeps scores times sqrt(hd), K then being log2 e / sqrt(hd).
constexpr float LOG2E = 1.4426950408889634f;
__device__ __forceinline__ float vezes(float m, float K) {
#pragma clang fp contract(off)
    return m * K;
}
__device__ __forceinline__ float peso(float s, float mL, float K = LOG2E) { return __builtin_amdgcn_exp2f(__builtin_fmaf(s, K, -mL)); }
// 2^(m K - M K) for m <= M, 0 where m is -inf (also M)
__device__ __forceinline__ float fator(float m, float M, float K = LOG2E) { return m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(vezes(m, K) - vezes(M, K)); }

template <int LPK>
__device__ __forceinline__ float soma_grupo(float v) {               // over LPK consecutive lanes, to all of them
    return [&] {
        auto dpp = [](float x, auto c) { return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), decltype(c)::value, 0xF, 0xF, false)); };
        if constexpr (LPK >= 2) v += dpp(v, std::integral_constant<int, 0xB1>{});
        if constexpr (LPK >= 4) v += dpp(v, std::integral_constant<int, 0x4E>{});
        if constexpr (LPK >= 8) v += dpp(v, std::integral_constant<int, 0x141>{});
        return v;
    }();
}
}  // namespace atc

// Exponent of a block of fp32 values in the int8 format, from the bits of the largest |v|, and the scale 2^-E: E = binary
// exponent - 7, one up where the largest mantissa rounds past 127 (half to even; products by 2^-E are exact). A block below
// 2^-126 is zero; one that holds an infinity or a NaN raises E_EXP and is zero.
__device__ __forceinline__ int expoente_f32(int bits, float& f, int kid, long long idx) {
    int E = (bits >> 23) - 133;
    f = __builtin_ldexpf(1.f, -E);
    if (__builtin_rintf(__int_as_float(bits) * f) > 127.f) { E++; f *= 0.5f; }
    if (bits >= 0x7f800000) reporta(E_EXP, kid, idx, E, bits);
    return E < -126 || bits >= 0x7f800000 ? E_ZERO : E;
}
// a block of LPB lanes x NV values to int8 mantissas; returns its exponent
template <int NV, int LPB>
__device__ __forceinline__ int quant_f32(const float (&v)[NV], int8_t (&q)[NV], int kid, long long idx0) {
    int bits = 0;
#pragma unroll
    for (int k = 0; k < NV; k++) bits = max(bits, __float_as_int(v[k]) & 0x7fffffff);
    float f;
    const int E = expoente_f32(g_max<LPB>(bits), f, kid, idx0);
#pragma unroll
    for (int k = 0; k < NV; k++) q[k] = E == E_ZERO ? 0 : (int8_t)(int)__builtin_rintf(v[k] * f);
    return E;
}

// 4 values of a row from position x on, as a block tensor (blocks of BLK values, whose lanes write together), bfloat16 or fp32
template <int BLK>
__device__ __forceinline__ void grava_4(void* out, int8_t* outE, int tipo, long long x, const float (&v)[4], int kid) {
    if (tipo == 0) {
        if constexpr (BLK >= 32) {
            int8_t q[4];
            const int E = quant_f32<4, BLK / 4>(v, q, kid, x);
            grava_i8<4, false>((int8_t*)out + x, q);
            if (x % BLK == 0) outE[x / BLK] = (int8_t)E;
        }
    } else if (tipo == 1) {
        typedef __bf16 b4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<b4*>((__bf16*)out + x) = b4{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
    } else {
        *reinterpret_cast<float4*>((float*)out + x) = make_float4(v[0], v[1], v[2], v[3]);
    }
}

// Joins the splits of a row and head, o = sum exp(m_s - m) o_s / sum exp(m_s - m) l_s (zeros for a row without visible
// tokens), and writes the row as a block tensor (TIPO 0), bfloat16 (1) or fp32 (2). NG groups of 32 threads share out the splits
// of 128 columns of a row, 4 columns a thread, four splits in flight at a time: one thread walking 64 splits one by one
// waited for each (30 us of a call of 131). With NG = 2 the groups are one wave, and a workgroup takes 512 columns in four of them;
// up to four splits (NG = 1) a wave takes 256 columns alone, there being nothing to share out.
template <int BLK, int TIPO, int NG>
__global__ void __launch_bounds__(NG <= 2 ? 256 : 32 * NG) k_atc_junta(const float* __restrict__ ml, const float* __restrict__ po, void* __restrict__ out,
                                                                       int8_t* __restrict__ oE, int C, int hd, int S, int kid) {
    constexpr int LC = NG == 1 ? 64 : 32;                             // lanes side by side along the columns
    const int r = blockIdx.x, ct = threadIdx.x % LC, g = threadIdx.x / LC % NG, faixa = NG <= 2 ? blockIdx.y * (blockDim.x >> 6) + (threadIdx.x >> 6) : blockIdx.y;
    const int col = faixa * 4 * LC + 4 * ct, cc = min(col, C - 4);
    const long long part = ((long long)r * (C / hd) + cc / hd) * S;
    const bool escrita = ml[2 * part + 1] < 0.f || col >= C;          // by its one split
    if (__all(escrita)) return;                                       // the waves that share splits have the same columns
    float M = -INFINITY, L = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = g; s0 < S; s0 += 4 * NG) {
        float2 x[4];
        float4 y[4];
        float mn = M;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int s = s0 + k * NG;
            x[k] = *reinterpret_cast<const float2*>(ml + 2 * (part + min(s, S - 1)));
            y[k] = *reinterpret_cast<const float4*>(po + (part + min(s, S - 1)) * hd + cc % hd);
            x[k].x = s < S ? x[k].x : -INFINITY;
            mn = fmaxf(mn, x[k].x);
        }
        const float al = atc::fator(M, mn);
        M = mn;
        L *= al;
#pragma unroll
        for (int d = 0; d < 4; d++) v[d] *= al;
#pragma unroll
        for (int k = 0; k < 4; k++) {                                 // a split without tokens has left its outputs unwritten
            const float f = atc::fator(x[k].x, M);
            const bool tem = f != 0.f || x[k].y != x[k].y;            // scores beyond fp32: f or the sum is NaN
            L += tem ? f * x[k].y : 0.f;
            v[0] += tem ? f * y[k].x : 0.f; v[1] += tem ? f * y[k].y : 0.f;
            v[2] += tem ? f * y[k].z : 0.f; v[3] += tem ? f * y[k].w : 0.f;
        }
    }
    if constexpr (NG == 1) {
        if (escrita) return;
    } else if constexpr (NG == 2) {
        const float MM = fmaxf(M, __shfl_xor(M, 32)), f = atc::fator(M, MM);
        L = L * f + __shfl_xor(L * f, 32);
#pragma unroll
        for (int d = 0; d < 4; d++) v[d] = v[d] * f + __shfl_xor(v[d] * f, 32);
        if (g > 0 || escrita) return;
    } else {
        __shared__ float sm[NG][32], sl[NG][32];
        __shared__ float4 sv[NG][32];
        sm[g][ct] = M;
        sl[g][ct] = L;
        sv[g][ct] = make_float4(v[0], v[1], v[2], v[3]);
        __syncthreads();
        if (g > 0 || escrita) return;
        float MM = M;
        for (int k = 1; k < NG; k++) MM = fmaxf(MM, sm[k][ct]);
        L = v[0] = v[1] = v[2] = v[3] = 0.f;
        for (int k = 0; k < NG; k++) {
            const float f = atc::fator(sm[k][ct], MM);
            const float4 x = sv[k][ct];
            L += f * sl[k][ct];
            v[0] += f * x.x; v[1] += f * x.y; v[2] += f * x.z; v[3] += f * x.w;
        }
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int k = 0; k < 4; k++) v[k] *= inv;
    grava_4<BLK>(out, oE, TIPO, (long long)r * C + col, v, kid);
}

namespace atc {
typedef __bf16 b8_t __attribute__((ext_vector_type(8)));
typedef short s4_t __attribute__((ext_vector_type(4)));
typedef float f4_t __attribute__((ext_vector_type(4)));
typedef int i4_t __attribute__((ext_vector_type(4)));
// The wait states an MFMA's result needs before another unit reads it, for results that more than one path reaches (the
// compiler counts them along one)
template <int N>
__device__ __forceinline__ void pronto(f4_t (&x)[N]) {
    static_assert(N == 1 || N == 2 || N == 4 || N == 8, "");
    if constexpr (N == 1) asm volatile("s_nop 7" : "+v"(x[0]));
    else if constexpr (N == 2) asm volatile("s_nop 7" : "+v"(x[0]), "+v"(x[1]));
    else if constexpr (N == 4) asm volatile("s_nop 7" : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]));
    else asm volatile("s_nop 7" : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]), "+v"(x[4]), "+v"(x[5]), "+v"(x[6]), "+v"(x[7]));
}

// A row without visible tokens: its outputs (or the marks of its split) for the query heads of kv head hk, by the whole
// workgroup
template <int HD>
__device__ __forceinline__ void vazia(const Args& a, long long r, int hk) {
    const int Gq = a.H / a.Hk, C = a.H * HD;
    for (int x = threadIdx.x; x < Gq * HD; x += blockDim.x) {
        const int h = hk * Gq + x / HD;
        const long long o = r * C + h * HD + x % HD;
        if (a.ml) {
            if (x % HD == 0) { float* y = a.ml + 2 * ((r * a.H + h) * a.S + blockIdx.z); y[0] = -INFINITY; y[1] = 0.f; }
        } else if (a.tipo == 0) {
            reinterpret_cast<int8_t*>(a.out)[o] = 0;
            if (!((h * HD + x % HD) & ((1 << a.lgblk) - 1))) a.outE[o >> a.lgblk] = E_ZERO;
        } else if (a.tipo == 1) reinterpret_cast<__bf16*>(a.out)[o] = (__bf16)0.f;
        else reinterpret_cast<float*>(a.out)[o] = 0.f;
    }
}

// Workgroup x as a tile of `por_wg` rows of a sequence: the sequences' tiles are numbered one after another, each sequence's last
// rows, which see the most keys, first. Every wave scans 64 sequences at a time. b = B past the last of the `total` tiles.
__device__ __forceinline__ void tile_de(const Args& a, int x, int por_wg, int& b, int& tile, int& total) {
    const int lane = threadIdx.x & 63, Gq = a.H / a.Hk;
    b = a.L.B;
    total = 0;
    for (int k = 0; k < a.L.B; k += 64) {
        const int s = min(k + lane, a.L.B - 1), n = a.L.ini ? a.L.ini[s + 1] - a.L.ini[s] : min(a.L.comp[s], 1);
        const int tiles = k + lane < a.L.B ? (int)(((long long)min(max(n, 0), a.L.M) * Gq + por_wg - 1) / por_wg) : 0;
        int ate = tiles;                                              // of this sequence and those before it
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int y = __shfl_up(ate, d);
            ate += lane >= d ? y : 0;
        }
        if (b == a.L.B && x < total + __shfl(ate, 63)) {
            const int q = __popcll(__ballot(total + ate <= x));
            b = k + q;
            tile = total + __shfl(ate, q) - 1 - x;
        }
        total += __shfl(ate, 63);
    }
}

// Rows r0 .. r0 + n - 1 of sequence b, comp tokens long; false (its rows, if any, zeroed) where it is malformed or has none. b = B:
// the rows of no sequence, every `passo`-th from `parte` on.
template <int HD>
__device__ __forceinline__ bool linhas_de(const Args& a, int b, bool primeiro, int parte, int passo, int hk, int& r0, int& n, int& comp) {
    if (b == a.L.B) {
        const int ini = a.L.ini ? a.L.ini[0] : 0, fim = a.L.ini ? a.L.ini[a.L.B] : a.L.B;
        for (long long x = parte; x < min(ini, a.L.M); x += passo) vazia<HD>(a, x, hk);
        for (long long x = max(fim, 0) + (long long)parte; x < a.L.M; x += passo) vazia<HD>(a, x, hk);
        return false;
    }
    if (!sequencia(a.L, b, r0, n, comp)) {
        const long long fim = a.L.ini ? (long long)a.L.ini[b + 1] : b + 1;
        if (primeiro)
            for (long long r = max(r0, 0); r < min(fim, (long long)a.L.M); r++) vazia<HD>(a, r, hk);
        return false;
    }
    if (!a.L.ini && n == 0 && primeiro && r0 < a.L.M) vazia<HD>(a, r0, hk);
    return n > 0;
}

// The tiles of TK keys that rows at positions i_lo .. i_hi see, numbered without gaps: those of the first tokens, then the
// window's; and this split's share of them
template <int TK>
struct Tiles {
    int lo, ns, nst, prim, t0, t1;
    bool uma;                                    // one split takes them all
    __device__ __forceinline__ Tiles(const Args& a, int i_lo, int i_hi) {
        lo = a.janela > 0 ? max(0, i_lo + 1 - a.janela) : 0;
        ns = min(a.sumid, lo);
        nst = (ns + TK - 1) / TK;
        prim = max(nst, lo / TK);
        const int T = nst + i_hi / TK - prim + 1;
        t0 = min((long long)blockIdx.z * a.fatia, (long long)T);
        t1 = min(t0 + a.fatia, T);
        uma = T <= a.fatia;
    }
    __device__ __forceinline__ int j0(int t) const { return TK * (t < nst ? t : t - nst + prim); }
};
// Whether some row sees key j of tile t
template <class T>
__device__ __forceinline__ bool visivel(const T& tl, int t, int j, int i_hi) { return (t < tl.t1) & (j <= i_hi) & ((j >= tl.lo) | (j < tl.ns)); }
// The page-table entry of key j (of some seen key where no row sees j). It is loaded a tile before it is used: whoever looks at it
// at once waits for every load issued before it, the tile's data among them.
__device__ __forceinline__ int entrada(const Args& a, int b, int j, int i_hi) { return a.L.tab[(long long)b * a.L.P + (min(j, i_hi) >> a.L.lgpag)]; }
// Entry p as a page to read from, whatever it holds (page 0 in place of one outside the cache): every load is made, without a
// branch, and a key that no row sees counts for nothing through its scale (escala). ok: whether the page is in the cache.
__device__ __forceinline__ int pagina(const Args& a, int p, bool& ok) {
    ok = (unsigned)p < (unsigned)a.L.npag;
    return ok ? p : 0;
}
__device__ __forceinline__ float escala(int E, bool conta) { return conta ? __builtin_ldexpf(1.f, E) : 0.f; }

// the bytes 32 k + 8 c .. + 7 of a head row: a lane's share of the k-th MFMA (zeros past the head's width)
template <int HD>
__device__ __forceinline__ long fragmento(const int8_t* linha, int k, int c) {
    if constexpr (HD >= 32) return *reinterpret_cast<const long*>(linha + 32 * k + 8 * c);
    else if constexpr (HD == 16) return c < 2 ? *reinterpret_cast<const long*>(linha + 8 * c) : 0;
    else return c == 0 ? (long)*reinterpret_cast<const unsigned*>(linha) : 0;
}

// A lane's query row: the MFMA operands, the scale of each exponent group, position, bias
template <int HD, int GS>
struct Linha {
    static constexpr int NM = HD < 32 ? 1 : HD / 32, G = HD / GS, MPG = NM / G;      // MFMAs of a score, groups, MFMAs of a group
    long q[NM];
    float fq[G], incl;
    long long r;
    int h, i;
    __device__ __forceinline__ Linha(const Args& a, int r0, int n, int comp, int hk, int rho, int c) {
        const int Gq = a.H / a.Hk, ld = (a.H + 2 * a.Hk) * HD;
        h = hk * Gq + rho % Gq;
        i = comp - n + rho / Gq;
        r = r0 + rho / Gq;
        incl = a.incl ? a.incl[h] : 0.f;
#pragma unroll
        for (int k = 0; k < NM; k++) q[k] = fragmento<HD>(a.qm + r * ld + h * HD, k, c);
#pragma unroll
        for (int g = 0; g < G; g++)
            fq[g] = __builtin_ldexpf(1.f / __builtin_sqrtf((float)HD), a.qE[r * (ld >> a.lgblk) + ((h * HD + g * GS) >> a.lgblk)]);
    }
    // scores of 16 keys (kf: their operands; f: 2^Ek per group of this lane's 4 keys 4 c ..), the first of which is j
    __device__ __forceinline__ void notas(const long (&kf)[NM], const float4 (&f)[G], int j, float* s) const {
        float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int g = 0; g < G; g++) {
            i4_t p = {0, 0, 0, 0};
#pragma unroll
            for (int k = g * MPG; k < (g + 1) * MPG; k++) p = __builtin_amdgcn_mfma_i32_16x16x32_i8(kf[k], q[k], p, 0, 0, 0);
            x[0] += (float)p[0] * (f[g].x * fq[g]); x[1] += (float)p[1] * (f[g].y * fq[g]);
            x[2] += (float)p[2] * (f[g].z * fq[g]); x[3] += (float)p[3] * (f[g].w * fq[g]);
        }
#pragma unroll
        for (int k = 0; k < 4; k++) s[k] = __builtin_fmaf(-incl, (float)(i - j) - (float)k, x[k]);   // distances below 2^24 are exact
    }
    __device__ __forceinline__ bool ve(const Args& a, int j) const { return (j <= i) & ((a.janela <= 0) | (j > i - a.janela) | (j < a.sumid)); }
};

// The running softmax of a lane's row and the outputs it accumulates, O^T tiles of 16 dimensions (lane: row, 4 dimensions)
template <int HD>
struct Corrente {
    static constexpr int DT = HD < 16 ? 1 : HD / 16;
    float m = -INFINITY, l = 0.f;
    f4_t o[DT];
    __device__ __forceinline__ Corrente() {
#pragma unroll
        for (int d = 0; d < DT; d++) o[d] = f4_t{0, 0, 0, 0};
    }
    // the maximum raised to a tile's scores s (4 keys of every 16 in a lane); returns what weights take off
    template <int N>
    __device__ __forceinline__ float sobe(const float (&s)[N], float K = LOG2E) {
        float mx = s[0];
#pragma unroll
        for (int k = 1; k < N; k++) mx = fmaxf(mx, s[k]);
        if (__any(mx > m + 7.2f / K)) {                               // 2^7.2: 5 nats; the exchange between lanes only then
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float mn = fmaxf(m, mx), al = fator(m, mn, K);
            m = mn;
            l *= al;
#pragma unroll
            for (int d = 0; d < DT; d++) o[d] *= al;
        }
        return m == -INFINITY ? 0.f : vezes(m, K);
    }
    // weights of 8 scores as three bf16 pieces, 24 bits, exactly
    __device__ __forceinline__ void pesos(const float* s, i4_t (&p)[3], float mL, float K = LOG2E) {
#pragma unroll
        for (int k = 0; k < 8; k += 2) {
            int y[3][2];
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const float e = peso(s[k + x], mL, K);
                l += e;
                y[0][x] = __float_as_int(e);
                const float e1 = e - __int_as_float(y[0][x] & 0xffff0000);
                y[1][x] = __float_as_int(e1);
                y[2][x] = __float_as_int(e1 - __int_as_float(y[1][x] & 0xffff0000));
            }
#pragma unroll
            for (int x = 0; x < 3; x++) p[x][k / 2] = (int)__builtin_amdgcn_perm((unsigned)y[x][1], (unsigned)y[x][0], 0x07060302u);
        }
    }
    __device__ __forceinline__ void soma_l() {
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
    }
    // the row's output, or its partial result. `uma`: this split is the row's only one; where blocks lie in a head the output is
    // then written here, and a negative sum tells the join so.
    template <int GS>
    __device__ __forceinline__ void grava(const Args& a, long long r, int h, int c, bool uma) {
        const int C = a.H * HD;
        const long long part = (r * a.H + h) * a.S + blockIdx.z;
        if (a.ml && uma && a.inteira) {
            if (blockIdx.z > 0) return;
            if (c == 0) a.ml[2 * part + 1] = -1.f;
        } else if (a.ml) {
            if (c == 0) { a.ml[2 * part] = m; a.ml[2 * part + 1] = l; }
            if (HD >= 16 || c == 0)
#pragma unroll
                for (int d = 0; d < DT; d++) *reinterpret_cast<f4_t*>(a.o + part * HD + 16 * d + 4 * c) = o[d];
            return;
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int d = 0; d < DT; d++) o[d] *= inv;
        const long long x = r * C + h * HD;
        if (a.tipo == 0) {                                            // blocks lie in the head (a plan's `direto`): GS = BLK
            if constexpr (HD >= 32) {
                constexpr int G = HD / GS, DG = DT / G;
#pragma unroll
                for (int g = 0; g < G; g++) {
                    int bits = 0;
#pragma unroll
                    for (int d = 0; d < 4 * DG; d++) bits = max(bits, __float_as_int(o[g * DG + d / 4][d % 4]) & 0x7fffffff);
                    bits = max(bits, __shfl_xor(bits, 16));
                    bits = max(bits, __shfl_xor(bits, 32));
                    float f;
                    const int E = expoente_f32(bits, f, a.kid, x + g * GS);
#pragma unroll
                    for (int d = g * DG; d < (g + 1) * DG; d++) {
                        int8_t z[4];
#pragma unroll
                        for (int k = 0; k < 4; k++) z[k] = E == E_ZERO ? 0 : (int8_t)(int)__builtin_rintf(o[d][k] * f);
                        grava_i8<4, false>((int8_t*)a.out + x + 16 * d + 4 * c, z);
                    }
                    if (c == 0) a.outE[(x >> a.lgblk) + g] = (int8_t)E;
                }
            }
        } else if (HD >= 16 || c == 0) {
#pragma unroll
            for (int d = 0; d < DT; d++) {
                typedef __bf16 b4_t __attribute__((ext_vector_type(4)));
                if (a.tipo == 1) *reinterpret_cast<b4_t*>((__bf16*)a.out + x + 16 * d + 4 * c) = b4_t{(__bf16)o[d][0], (__bf16)o[d][1], (__bf16)o[d][2], (__bf16)o[d][3]};
                else *reinterpret_cast<f4_t*>((float*)a.out + x + 16 * d + 4 * c) = o[d];
            }
        }
    }
};

// O^T += V^T P^T over 32 keys, whose values are the rows of v in LDS (VS bf16 each) and whose weights are p
template <int HD, int VS>
__device__ __forceinline__ void soma_v(Corrente<HD>& y, const __bf16* v, const i4_t (&p)[3], int lr, int c) {
    typedef __attribute__((address_space(3))) s4_t* lds4;
    constexpr int DT = Corrente<HD>::DT, DB = DT < 4 ? DT : 4;        // four tiles of dimensions at a time: products in a row do not wait for one another
#pragma unroll
    for (int d0 = 0; d0 < DT; d0 += DB) {
        b8_t x[DB];
#pragma unroll
        for (int d = 0; d < DB; d++) {
            // lane 16 c + x reads row 4 c + x / 4, columns 4 (x % 4) ..; it receives column x of the 4 rows
            const __bf16* z = v + (4 * c + lr / 4) * VS + 16 * (d0 + d) + 4 * (lr % 4);
            const s4_t v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(z)), v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(z + 16 * VS));
            x[d] = __builtin_bit_cast(b8_t, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
        }
#pragma unroll
        for (int k = 0; k < 3; k++)
#pragma unroll
            for (int d = 0; d < DB; d++) y.o[d0 + d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[d], __builtin_bit_cast(b8_t, p[k]), y.o[d0 + d], 0, 0, 0);
    }
    pronto(y.o);
}

// VB mantissas of a value and its exponent, into a row of bf16 in LDS: m 2^E is exact there. A row narrower than 16 is
// filled up with zeros.
template <int VB>
__device__ __forceinline__ void valor_lds(__bf16* p, const int4& d, float e) {
    const int y[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
    for (int k = 0; k < 16; k += 8) {
        b8_t z;
#pragma unroll
        for (int x = 0; x < 8; x++) z[x] = (__bf16)(k + x < VB ? e * (float)(int8_t)(y[(k + x) / 4] >> (8 * (x % 4))) : 0.f);
        *reinterpret_cast<b8_t*>(p + k) = z;
    }
}
template <int VB>
__device__ __forceinline__ int4 le_vb(const int8_t* p) {
    if constexpr (VB == 16) return *reinterpret_cast<const int4*>(p);
    else return make_int4(*reinterpret_cast<const int*>(p), 0, 0, 0);
}
}  // namespace atc

// One row (token, query head) and one split of its visible tokens per workgroup, the four waves a tile of 4 wave loads each in
// turn. Softmax in one pass: every group of LPK lanes (a key's head row, 16 bytes a lane) keeps the running maximum m, sum l and
// output o of the keys it has seen,
//   u = 2^(Eq + Ek) (mq . mk) / sqrt(hd) - incl (i - j);  p = exp(u - m);  o += p 2^Ev mv,
// and they are joined at the end (lanes, waves, then the splits by k_atc_junta). Products of mantissas are exact in int32
// (v_dot4), statistics and outputs fp32. Only the page table is read a tile ahead: holding the next tile's bytes too costs a fifth
// of the waves and is slower (104 us against 92 below).
// Reading the keys and values bounds it: 4 sequences of 90,001 to 131,071 tokens, 8 heads of 64 take 94 us, 4.97 TB/s of cache (a
// large copy reaches 5.5). Short contexts are latency: one of 200 tokens 6.7 us, the launch and three round trips to memory.
template <int HD, int GS>
__global__ void __launch_bounds__(256) k_atc_um(atc::Args a) {
    using namespace atc;
    constexpr int VB = HD < 16 ? HD : 16, LPK = HD / VB, KPW = 64 / LPK, U = 4, NW = 4, G = HD / GS, TK = U * KPW;
    constexpr bool UMA = KPW <= 16;                                   // a wave load's keys lie in one page
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = lane % LPK;
    const int r = blockIdx.x, h = blockIdx.y, hk = h / (a.H / a.Hk), g = c * VB / GS, pag = 1 << a.L.lgpag;
    const Seq q = acha(a.L, r);
    Tiles<TK> tl(a, max(q.i, 0), max(q.i, 0));
    if (!q.ok) { tl.t0 = tl.t1 = 0; tl.uma = true; }

    int qv[VB / 4];
    const int ld = (a.H + 2 * a.Hk) * HD, col = h * HD + c * VB;
#pragma unroll
    for (int k = 0; k < VB / 4; k++) qv[k] = reinterpret_cast<const int*>(a.qm + (long long)r * ld + col)[k];
    const int eq = a.qE[(long long)r * (ld >> a.lgblk) + (col >> a.lgblk)];
    const float esc = 1.f / __builtin_sqrtf((float)HD), incl = a.incl ? a.incl[h] : 0.f;

    const long long dv = (long long)a.Hk * pag;                       // slots between a token's key and its value
    int pg[U], p0[U], kv[U][VB / 4], vv[U][VB / 4], ruim = -1;
    int8_t ek[U], ev[U];
    bool ok[U];
    auto chave = [&](int t, int u) { return tl.j0(t) + u * KPW + lane / LPK; };
    auto le_paginas = [&](int t) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int j = chave(min(t, tl.t1 - 1), u);
            pg[u] = entrada(a, q.b, UMA ? __builtin_amdgcn_readfirstlane(j) : j, q.i);
        }
    };
    auto acha_paginas = [&](int t) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            p0[u] = pagina(a, UMA ? __builtin_amdgcn_readfirstlane(pg[u]) : pg[u], ok[u]);
            const int j = chave(t, u);
            ruim = !ok[u] && visivel(tl, t, j, q.i) ? j : ruim;
        }
    };
    auto vaga = [&](int t, int u) { return (long long)hk * pag + (chave(t, u) & (pag - 1)); };
    auto le_chaves = [&](int t) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int8_t* m = a.cm + p0[u] * a.pag_m + vaga(t, u) * HD + c * VB;
#pragma unroll
            for (int k = 0; k < VB / 4; k++) kv[u][k] = reinterpret_cast<const int*>(m)[k];
            ek[u] = a.cE[p0[u] * a.pag_e + vaga(t, u) * G + g];
        }
    };
    auto le_valores = [&](int t) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int8_t* m = a.cm + p0[u] * a.pag_m + (dv + vaga(t, u)) * HD + c * VB;
#pragma unroll
            for (int k = 0; k < VB / 4; k++) vv[u][k] = reinterpret_cast<const int*>(m)[k];
            ev[u] = a.cE[p0[u] * a.pag_e + (dv + vaga(t, u)) * G + g];
        }
    };

    float m = -INFINITY, l = 0.f, o[VB];
#pragma unroll
    for (int d = 0; d < VB; d++) o[d] = 0.f;
    int t = tl.t0 + w;
    if (t < tl.t1) le_paginas(t);
    for (; t < tl.t1; t += NW) {
        const int j0 = tl.j0(t);
        acha_paginas(t);
        le_chaves(t);
        le_valores(t);
        le_paginas(t + NW);
        const bool cheia = (j0 + TK - 1 <= q.i) & ((j0 >= tl.lo) | (j0 + TK <= tl.ns));
        float s[U], mn = m;
        bool vis[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int j = chave(t, u);
            vis[u] = ok[u] & (cheia | visivel(tl, t, j, q.i));
            int d = 0;
#pragma unroll
            for (int k = 0; k < VB / 4; k++) d = __builtin_amdgcn_sdot4(qv[k], kv[u][k], d, false);
            s[u] = soma_grupo<LPK>(__builtin_ldexpf((float)d, eq + ek[u])) * esc - incl * (float)(q.i - j);
            s[u] = vis[u] ? s[u] : -INFINITY;
            mn = fmaxf(mn, s[u]);
        }
        if (__any(mn > m)) {
            const float al = fator(m, mn);
            m = mn;
            l *= al;
#pragma unroll
            for (int d = 0; d < VB; d++) o[d] *= al;
        }
        const float mL = m == -INFINITY ? 0.f : vezes(m, LOG2E);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const float e = peso(s[u], mL), pv = vis[u] ? __builtin_ldexpf(e, ev[u]) : 0.f;
            l += e;
#pragma unroll
            for (int d = 0; d < VB; d++) o[d] += pv * (float)(int8_t)(vv[u][d / 4] >> (8 * (d % 4)));
        }
    }
    relata_pagina(a, q.b, ruim);

    // the wave's groups: a common maximum, then sums in which every step halves the values a lane still holds
    float M = m;
#pragma unroll
    for (int x = LPK; x < 64; x *= 2) M = fmaxf(M, __shfl_xor(M, x));
    const float es = fator(m, M);
    l *= es;
#pragma unroll
    for (int x = LPK; x < 64; x *= 2) l += __shfl_xor(l, x);
#pragma unroll
    for (int d = 0; d < VB; d++) o[d] *= es;
    int d0 = 0;
#pragma unroll
    for (int x = LPK, n = VB; x < 64; x *= 2) {
        if (n > 1) {
            n /= 2;
            const bool alto = lane & x;
#pragma unroll
            for (int d = 0; d < VB / 2; d++)
                if (d < n) {
                    const float fica = alto ? o[d + n] : o[d], vai = alto ? o[d] : o[d + n];
                    o[d] = fica + __shfl_xor(vai, x);
                }
            d0 += alto ? n : 0;
        } else o[0] += __shfl_xor(o[0], x);
    }
    constexpr int RESTO = VB / KPW > 1 ? VB / KPW : 1;                // values a lane is left with
    __shared__ __align__(16) float so[NW][HD];
    __shared__ float sm[NW], sl[NW];
#pragma unroll
    for (int d = 0; d < RESTO; d++) so[w][c * VB + d0 + d] = o[d];    // lanes with the same values write the same
    if (lane == 0) { sm[w] = M; sl[w] = l; }
    __syncthreads();
    if (threadIdx.x >= HD / 4) {
        if (r == 0 && h == 0 && blockIdx.z == 0) confere(a.L, a.kid, threadIdx.x - HD / 4, 256 - HD / 4);
        return;
    }
    float MM = sm[0], LL = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 1; k < NW; k++) MM = fmaxf(MM, sm[k]);
#pragma unroll
    for (int k = 0; k < NW; k++) {
        const float f = fator(sm[k], MM);
        const float4 x = *reinterpret_cast<const float4*>(&so[k][4 * threadIdx.x]);
        LL += sl[k] * f;
        v[0] += f * x.x; v[1] += f * x.y; v[2] += f * x.z; v[3] += f * x.w;
    }
    const long long part = ((long long)r * a.H + h) * a.S + blockIdx.z;
    if (a.ml && !(tl.uma && a.inteira)) {
        *reinterpret_cast<float4*>(a.o + part * HD + 4 * threadIdx.x) = make_float4(v[0], v[1], v[2], v[3]);
        if (threadIdx.x == 0) { a.ml[2 * part] = MM; a.ml[2 * part + 1] = LL; }
        return;
    }
    if (a.ml) {                                                       // the row's one split: written here
        if (blockIdx.z > 0) return;
        if (threadIdx.x == 0) a.ml[2 * part + 1] = -1.f;
    }
    const float inv = LL == 0.f ? 0.f : 1.f / LL;
#pragma unroll
    for (int k = 0; k < 4; k++) v[k] *= inv;
    grava_4<GS>(a.out, a.outE, a.tipo, (long long)r * a.H * HD + h * HD + 4 * threadIdx.x, v, a.kid);
}

// Many rows that share keys and values (new tokens of a sequence, query heads of a group): 16 a wave, 64 per workgroup, on
// matrix cores; the workgroup walks its keys in tiles of 64. Row rho of a (sequence, kv head) is token rho / Gq,
// head rho % Gq of the group.
//   What bounds it is the VALU (0.94 busy): some 440 instructions per wave and tile of 16 rows x 64 keys, of which the weights' powers,
// sums and pieces are 140, the scores and their maximum 60, the tile's staging 90. 8 prompts of 1 to 4000 tokens, 8 heads of 64:
// 184 us with the join and the output's values, 254 TFLOP/s; their matrix products alone 39 us. Heads of up to 64 fit four waves a SIMD
// (128 registers): the pieces of 32 keys are made and used before the next 32's (three waves, all 64 keys' pieces at once: 193 us).
// Weights summed by matrix products with ones instead of additions: 192 us.
//   S^T = K Q^T by bf16 MFMA on the values m 2^E themselves, exact in bf16 (8 bits), sums in fp32: a lane holds one row (lane %
//   16) and 4 keys of each 16, so maxima and sums are in-lane but for two exchanges, and P^T is the next product's
//   operand as it stands. (i8 MFMA, exact, costs a conversion and two products per score and exponent group: 281 us for
//   these prompts, 210 this way.)
//   O^T = V^T P^T by bf16 MFMA: P is three bf16 pieces, exact (one piece would leave 2^-8 of every weight, two 2^-16). V^T
//   comes from row-major LDS by transposing reads.
// Keys and values are staged once per workgroup, two tiles in LDS: the next tile's loads are in flight while this one is
// computed, its page numbers one tile earlier still. Slots no row sees are staged as zeros, whatever they hold. The running maximum is
// raised (and O rescaled) only where a tile exceeds it by 5 nats: weights are then at most e^5, which costs fp32 no precision.
template <int HD, int GS>
__global__ void __launch_bounds__(256, HD <= 64 ? 4 : 2) k_atc_mf(atc::Args a) {
    using namespace atc;
    constexpr int VB = HD < 16 ? HD : 16, LPK = HD / VB, G = HD / GS, TK = 64, NM = HD < 32 ? 1 : HD / 32, RW = 64;
    constexpr int VS = 16 * Corrente<HD>::DT + 8;                     // LDS rows, in values; keys and values alike
    constexpr int NT = TK * LPK, IT = (NT + 255) / 256; // staging: chunks of a tile's keys (and of its values), per thread
    __shared__ __align__(16) __bf16 sk[2][TK * VS], sv[2][TK * VS];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, lr = lane & 15, c = lane >> 4, hk = blockIdx.y, Gq = a.H / a.Hk;
    if (blockIdx.x == gridDim.x - 1 && hk == 0 && blockIdx.z == 0) confere(a.L, a.kid, threadIdx.x, 256);
    int b, tile = 0, total, r0, n, comp;
    tile_de(a, blockIdx.x, RW, b, tile, total);
    if (!linhas_de<HD>(a, b, tile == 0, blockIdx.x - total, gridDim.x - total, hk, r0, n, comp)) return;
    const int linhas = n * Gq, rho0 = tile * RW, i_lo = comp - n + rho0 / Gq, i_hi = comp - n + min(rho0 + RW - 1, linhas - 1) / Gq;
    const Tiles<TK> tl(a, i_lo, i_hi);
    const int rho = rho0 + 16 * w + lr, w_hi = comp - n + min(rho0 + 16 * w + 15, linhas - 1) / Gq;   // w_hi: the wave's last position
    const bool tem = rho0 + 16 * w < linhas;

    // this lane's query row as MFMA operands: m 2^E in bf16, exact
    const int rc = min(rho, linhas - 1), h = hk * Gq + rc % Gq, i = comp - n + rc / Gq, ld = (a.H + 2 * a.Hk) * HD;
    const long long r = r0 + rc / Gq;
    const float raiz = __builtin_sqrtf((float)HD), K = LOG2E / raiz, incl = a.incl ? a.incl[h] * raiz : 0.f;
    b8_t q[NM];
#pragma unroll
    for (int k = 0; k < NM; k++) {
        const long x = fragmento<HD>(a.qm + r * ld + h * HD, k, c);
        const int col = h * HD + (HD >= 32 ? 32 * k + 8 * c : 0);
        const float e = __builtin_ldexpf(1.f, a.qE[r * (ld >> a.lgblk) + (col >> a.lgblk)]);
#pragma unroll
        for (int z = 0; z < 8; z++) q[k][z] = (__bf16)(e * (float)(int8_t)(x >> (8 * z)));
    }

    // Staging: a thread's chunks of VB bytes, key `chave` and its value. A tile's 16 keys 16 x .. lie in one page (pages hold 16 or
    // more), so where a wave's keys do too its entry is one scalar read.
    const int pag = 1 << a.L.lgpag, cc = threadIdx.x % LPK;
    const long long dvm = (long long)a.Hk * pag * HD, dve = (long long)a.Hk * pag * G;        // from a key to its value
    constexpr bool UMA = 64 / LPK <= 16;
    int pg[IT], ruim = -1;
    int8_t de[2][IT];
    int4 dm[2][IT];
    bool conta[IT];
    auto chave = [&](int x) { return min((int)(threadIdx.x + 256 * x) / LPK, TK - 1); };
    auto le_paginas = [&](int t) {
#pragma unroll
        for (int x = 0; x < IT; x++) {
            const int j = tl.j0(min(t, tl.t1 - 1)) + chave(x);
            pg[x] = entrada(a, b, UMA ? __builtin_amdgcn_readfirstlane(j) : j, i_hi);
        }
    };
    auto le_dados = [&](int t) {
#pragma unroll
        for (int x = 0; x < IT; x++) {
            const int j = tl.j0(t) + chave(x);
            bool ok;
            const int p = pagina(a, UMA ? __builtin_amdgcn_readfirstlane(pg[x]) : pg[x], ok);
            const bool vis = visivel(tl, t, j, i_hi);
            ruim = vis && !ok ? j : ruim;
            conta[x] = vis && ok;
            const long long vaga = (long long)hk * pag + (j & (pag - 1));
            const int8_t *m = a.cm + p * a.pag_m + vaga * HD + cc * VB, *e = a.cE + p * a.pag_e + vaga * G + cc * VB / GS;
            dm[0][x] = le_vb<VB>(m);
            dm[1][x] = le_vb<VB>(m + dvm);
            de[0][x] = e[0];
            de[1][x] = e[dve];
        }
    };
    auto guarda = [&](int buf) {
#pragma unroll
        for (int x = 0; x < IT; x++) {
            if ((int)threadIdx.x + 256 * x >= NT) continue;
            const int o = chave(x) * VS + cc * VB;
            valor_lds<VB>(&sk[buf][o], dm[0][x], escala(de[0][x], conta[x]));
            valor_lds<VB>(&sv[buf][o], dm[1][x], escala(de[1][x], conta[x]));
        }
    };

    Corrente<HD> y;
    if (tl.t0 < tl.t1) {
        le_paginas(tl.t0);
        le_dados(tl.t0);
        le_paginas(tl.t0 + 1);
        guarda(0);
    }
    __syncthreads();
    for (int t = tl.t0; t < tl.t1; t++) {
        const int buf = (t - tl.t0) & 1, j0 = tl.j0(t);
        if (t + 1 < tl.t1) { le_dados(t + 1); le_paginas(t + 2); }
        if (tem && j0 <= w_hi) {
            f4_t x[4];
            const float bias = -incl * (float)(i - j0 - 4 * c);       // the product starts from the bias of each key
#pragma unroll
            for (int k = 0; k < 16; k++) x[k / 4][k % 4] = __builtin_fmaf(incl, (float)(16 * (k / 4) + k % 4), bias);
#pragma unroll
            for (int kt = 0; kt < 4; kt++)
#pragma unroll
                for (int k = 0; k < NM; k++) {
                    b8_t kf = b8_t{};
                    if (HD >= 32 || c < 2) kf = *reinterpret_cast<const b8_t*>(&sk[buf][(16 * kt + lr) * VS + 32 * k + 8 * c]);
                    x[kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, q[k], x[kt], 0, 0, 0);
                }
            pronto(x);
            float s[16];
#pragma unroll
            for (int k = 0; k < 16; k++) s[k] = x[k / 4][k % 4];
            // where every key of the tile is visible to every row of the workgroup there is nothing to mask
            if (j0 + TK - 1 > i_lo || (a.janela > 0 && j0 <= i_hi - a.janela && j0 + TK > a.sumid)) {
                const int janela = a.janela > 0 ? a.janela : 0x7fffffff;
#pragma unroll
                for (int k = 0; k < 16; k++) {
                    const int j = j0 + 4 * c + 16 * (k / 4) + k % 4;
                    s[k] = (j <= i) & ((i - j < janela) | (j < a.sumid)) ? s[k] : -INFINITY;
                }
            }
            const float mL = y.sobe(s, K);
#pragma unroll
            for (int kk = 0; kk < 2; kk++) {
                i4_t p[3];
                y.pesos(s + 8 * kk, p, mL, K);
                soma_v<HD, VS>(y, &sv[buf][32 * kk * VS], p, lr, c);
            }
        }
        if (t + 1 < tl.t1) guarda(buf ^ 1);
        __syncthreads();
    }
    if (hk == 0) relata_pagina(a, b, ruim);
    if (rho >= linhas) return;
    y.soma_l();
    y.m *= 1.f / raiz;                                                // in nats, as the join takes it
    y.template grava<GS>(a, r, h, c, tl.uma);
}

// Up to 16 rows that share keys and values (a new token's query heads of a group, a few new tokens): the same products, but the
// four waves of a workgroup take every fourth tile of 32 keys for the same rows, without a barrier. A wave reads its keys
// from memory in the MFMA's own layout, passes its values through its own LDS to transpose them, and has the next
// tile's bytes in flight while it computes this one. The waves' results are joined at the end.
// Reading the keys and values bounds it, at 2 waves per SIMD (196 registers; held to 168, which would make them 3, it spills: 155 us): 64
// sequences of 500 to 4096 tokens, 32 query heads on 8 of 128, 88 us, 3.5 TB/s; 126 us with loads issued when they are needed.
template <int HD, int GS>
__global__ void __launch_bounds__(256) k_atc_gr(atc::Args a) {
    using namespace atc;
    constexpr int VB = HD < 16 ? HD : 16, LPK = HD / VB, G = HD / GS, TK = 32, NM = Linha<HD, GS>::NM, DT = Corrente<HD>::DT;
    constexpr int VS = 16 * DT + 8, IT = (TK * LPK + 63) / 64;
    constexpr int BV = TK * VS * 2, BF = G * TK * 4, BO = 3 * DT * 64 * 16, BYTES = 4 * (BV + BF) > BO ? 4 * (BV + BF) : BO;
    __shared__ __align__(16) char mem[BYTES];                         // per wave: values, key scales; at the end the waves' outputs
    __shared__ float sm[4][16], sl[4][16];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, lr = lane & 15, c = lane >> 4, hk = blockIdx.y, Gq = a.H / a.Hk;
    __bf16* sv = reinterpret_cast<__bf16*>(mem + w * (BV + BF));
    float* sf = reinterpret_cast<float*>(mem + w * (BV + BF) + BV);
    if (blockIdx.x == gridDim.x - 1 && hk == 0 && blockIdx.z == 0) confere(a.L, a.kid, threadIdx.x, 256);
    int r0, n, comp;
    if (!linhas_de<HD>(a, blockIdx.x, true, 0, 1, hk, r0, n, comp)) return;
    const int b = blockIdx.x, linhas = n * Gq, i_lo = comp - n, i_hi = comp - 1, pag = 1 << a.L.lgpag;
    const Tiles<TK> tl(a, i_lo, i_hi);
    const Linha<HD, GS> q(a, r0, n, comp, hk, min(lr, linhas - 1), c);

    // The tile's first and second 16 keys lie in one page each: two scalar table reads. A lane's keys: lr and 16 + lr for the
    // products; lane / LPK, then 64 / LPK further on, for the values. Keys are read again once the products have taken them, values
    // once they are in LDS.
    constexpr int KV = 64 / LPK;
    int pg[2], p0[2], ruim = -1;
    int8_t ke[2], ve[IT];
    bool ok[2];
    long kf[2][NM];
    int4 dv[IT];
    auto le_paginas = [&](int t) {
#pragma unroll
        for (int k = 0; k < 2; k++) pg[k] = entrada(a, b, __builtin_amdgcn_readfirstlane(tl.j0(min(t, tl.t1 - 1)) + 16 * k), i_hi);
    };
    auto acha_paginas = [&](int t) {
#pragma unroll
        for (int k = 0; k < 2; k++) {
            p0[k] = pagina(a, __builtin_amdgcn_readfirstlane(pg[k]), ok[k]);
            const int j = tl.j0(t) + 16 * k + lr;
            ruim = !ok[k] && visivel(tl, t, j, i_hi) ? j : ruim;
        }
    };
    auto vaga = [&](int t, int key) { return (long long)hk * pag + ((tl.j0(t) + key) & (pag - 1)); };
    auto le_chaves = [&](int t) {
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const long long v = vaga(t, 16 * k + lr);
#pragma unroll
            for (int x = 0; x < NM; x++) kf[k][x] = fragmento<HD>(a.cm + p0[k] * a.pag_m + v * HD, x, c);
            ke[k] = a.cE[p0[k] * a.pag_e + v * G + min(c, G - 1)];
        }
    };
    auto le_valores = [&](int t) {
#pragma unroll
        for (int x = 0; x < IT; x++) {
            const int key = min(lane / LPK + KV * x, TK - 1), cc = lane % LPK, p = KV <= 16 ? p0[KV * x / 16] : key < 16 ? p0[0] : p0[1];
            const long long v = (long long)a.Hk * pag + vaga(t, key);
            dv[x] = le_vb<VB>(a.cm + p * a.pag_m + v * HD + cc * VB);
            ve[x] = a.cE[p * a.pag_e + v * G + cc * VB / GS];
        }
    };

    Corrente<HD> y;
    int t = tl.t0 + w;
    if (t < tl.t1) {
        le_paginas(t);
        acha_paginas(t);
        le_chaves(t);
        le_valores(t);
        le_paginas(t + 4);
    }
    for (; t < tl.t1; t += 4) {
        const int j0 = tl.j0(t), prox = min(t + 4, tl.t1 - 1);
        const bool cheia = j0 + TK - 1 <= i_hi && (j0 >= tl.lo || j0 + TK <= tl.ns);          // some row sees each of its keys
#pragma unroll
        for (int k = 0; k < 2; k++)
            if (c < G) sf[c * TK + 16 * k + lr] = escala(ke[k], ok[k] & (cheia | visivel(tl, t, j0 + 16 * k + lr, i_hi)));
#pragma unroll
        for (int x = 0; x < IT; x++) {
            const int key = lane / LPK + KV * x;
            const bool bom = KV <= 16 ? ok[KV * x / 16 % 2] : key < 16 ? ok[0] : ok[1];
            if (key < TK) valor_lds<VB>(sv + key * VS + lane % LPK * VB, dv[x], escala(ve[x], bom & (cheia | visivel(tl, t, j0 + key, i_hi))));
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        acha_paginas(prox);
        le_valores(prox);
        float s[8];
#pragma unroll
        for (int k = 0; k < 2; k++) {
            float4 f[G];
#pragma unroll
            for (int g = 0; g < G; g++) f[g] = *reinterpret_cast<const float4*>(sf + g * TK + 16 * k + 4 * c);
            q.notas(kf[k], f, j0 + 16 * k + 4 * c, s + 4 * k);
        }
        le_chaves(prox);
        le_paginas(t + 8);
        if (j0 + TK - 1 > i_lo || (a.janela > 0 && j0 <= i_hi - a.janela && j0 + TK > a.sumid)) {
#pragma unroll
            for (int k = 0; k < 8; k++) s[k] = q.ve(a, j0 + 16 * (k / 4) + 4 * c + k % 4) ? s[k] : -INFINITY;
        }
        i4_t p[3];
        y.pesos(s, p, y.sobe(s));
        soma_v<HD, VS>(y, sv, p, lr, c);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    relata_pagina(a, b, ruim);
    // the four waves' results: a common maximum, then sums
    y.soma_l();
    if (c == 0) { sm[w][lr] = y.m; sl[w][lr] = y.l; }
    __syncthreads();
    float M = sm[0][lr], L = 0.f;
#pragma unroll
    for (int k = 1; k < 4; k++) M = fmaxf(M, sm[k][lr]);
#pragma unroll
    for (int k = 0; k < 4; k++) L += sl[k][lr] * fator(sm[k][lr], M);
    const float f = fator(y.m, M);
    f4_t* so = reinterpret_cast<f4_t*>(mem);
#pragma unroll
    for (int d = 0; d < DT; d++) {
        y.o[d] *= f;
        if (w > 0) so[((w - 1) * DT + d) * 64 + lane] = y.o[d];
    }
    __syncthreads();
    if (w > 0 || lr >= linhas) return;
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int k = 0; k < 3; k++) y.o[d] += so[(k * DT + d) * 64 + lane];
    y.m = M;
    y.l = L;
    y.template grava<GS>(a, q.r, q.h, c, tl.uma);
}

// ---------------------------------------------------------------------------------------------- values
// A block or raw tensor as floats (the inverse of de_f32), each value rounded once: block values are exact in both types
// (8 bits), raw ones are scaled in double precision and rounded to fp32. 8 values a lane; bound by its bytes: 16,000 x 512 to
// bf16 5.3 us, 4.7 TB/s.
template <int TIPO>
__global__ void __launch_bounds__(256) k_valores(const int8_t* __restrict__ m, const int8_t* __restrict__ E, void* __restrict__ out, long long n, int lgblk) {
    const long long o = ((long long)blockIdx.x * 256 + threadIdx.x) * 8;
    if (o >= n) return;
    int v[8];
    le_i8(m + o, v);
    const int e = E[o >> lgblk];
    if constexpr (TIPO == 1) {
        typedef __bf16 b8 __attribute__((ext_vector_type(8)));
        b8 y;
#pragma unroll
        for (int k = 0; k < 8; k++) y[k] = (__bf16)__builtin_ldexpf((float)v[k], e);
        *reinterpret_cast<b8*>((__bf16*)out + o) = y;
    } else {
        float4* y = reinterpret_cast<float4*>((float*)out + o);
#pragma unroll
        for (int k = 0; k < 2; k++)
            y[k] = make_float4(__builtin_ldexpf((float)v[4 * k], e), __builtin_ldexpf((float)v[4 * k + 1], e),
                               __builtin_ldexpf((float)v[4 * k + 2], e), __builtin_ldexpf((float)v[4 * k + 3], e));
    }
}
__global__ void __launch_bounds__(256) k_valores_cru(const int* __restrict__ acc, const int16_t* __restrict__ e, float* __restrict__ out, long long n) {
    const long long o = (long long)blockIdx.x * 256 + threadIdx.x;
    if (o < n) out[o] = (float)__builtin_ldexp((double)acc[o], e[o]);
}
