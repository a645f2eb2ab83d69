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

// first row, row count and length of sequence b; false (and E_ARG, from the one lane that asks) where they are malformed
__device__ __forceinline__ bool sequencia(const Lote& L, int b, int& r0, int& n, int& comp, int kid, bool relata) {
    comp = L.comp[b];
    r0 = L.ini ? L.ini[b] : b;
    n = L.ini ? L.ini[b + 1] - r0 : min(comp, 1);                     // without starts, an empty sequence has no row
    const bool ok = r0 >= 0 && n >= 0 && r0 <= L.M - n && n <= L.novos && comp >= n && comp <= L.teto;
    if (!ok && relata) reporta(E_ARG, kid, r0, comp, b);
    return ok;
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

__device__ __forceinline__ Seq acha(const Lote& L, int r, int kid, bool relata) {
    Seq s{sequencia_de(L, r), 0, 0};
    if (s.b < 0) return s;
    int r0, n, comp;
    s.ok = sequencia(L, s.b, r0, n, comp, kid, relata);
    s.ok = s.ok && r - r0 < n;
    s.i = comp - n + (r - r0);
    return s;
}
}  // namespace atc

// ---------------------------------------------------------------------------------------------- pages
// The rows' keys and values into their slots. A thread moves VB bytes (a head's 16, or its 4): the threads of a wave hold
// the same chunks of consecutive rows, whose slots are consecutive, so a wave writes whole kilobytes of a page's tile.
// Bound by its bytes, read and written once.
template <int HD, int GS>
__global__ void __launch_bounds__(256) k_cache_grava(const int8_t* __restrict__ qm, const int8_t* __restrict__ qE, int8_t* __restrict__ cm,
                                                     int8_t* __restrict__ cE, atc::Lote L, int H, int Hk, int lgblk, long long pag_m,
                                                     long long pag_e, int kid) {
    constexpr int VB = HD < 16 ? HD : 16, NC = HD / VB, G = HD / GS, LPW = 64 / NC;     // LPW: rows per wave
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int r = blockIdx.x * LPW + lane / NC, c = lane % NC;
    const int kvh = blockIdx.y * 4 + w;                                                 // keys' heads, then values'
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
    if (!atc::sequencia(L, b, r0, n, comp, kid, kvh == 0 && c == 0) || r - r0 >= n) return;
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
// keeps them). The pairs' targets are distinct and no pair's source, which the host has checked.
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
    float *ml, *o;                               // partial results: (maximum, sum) and outputs per (row, head, split)
    long long pag_m, pag_e;
    Lote L;
    int H, Hk, lgblk, janela, sumid, S, fatia, kid;   // S splits of `fatia` visible tokens each
};

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

// One row (token, query head) and one split of its visible tokens per workgroup. Softmax in one pass: every group of LPK
// lanes (a key's head row, 16 bytes a lane) keeps the running maximum m, sum l and output o of the keys it has seen,
//   u = 2^(Eq + Ek) (mq . mk) / sqrt(hd) - incl (i - j), in units of log2 e;  p = 2^(u - m);  o += p 2^Ev mv,
// and they are joined at the end (lanes, waves, then the splits by k_atc_junta). Products of mantissas are exact in int32
// (v_dot4), statistics and outputs fp32. The visible tokens are numbered x = 0 .. nvis - 1 without gaps, the first tokens
// then the window, so no masked key is read.
template <int HD, int GS>
__global__ void __launch_bounds__(256) k_atc_um(atc::Args a) {
    constexpr int VB = HD < 16 ? HD : 16, LPK = HD / VB, KPW = 64 / LPK, U = 4, NW = 4, G = HD / GS;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = lane % LPK;
    const int r = blockIdx.x, h = blockIdx.y, s = blockIdx.z, hk = h / (a.H / a.Hk), g = c * VB / GS;
    const atc::Seq q = atc::acha(a.L, r, a.kid, threadIdx.x == 0 && h == 0 && s == 0);
    int nvis = 0, ns = 0, lo = 0;
    if (q.ok) {
        lo = a.janela > 0 ? max(0, q.i + 1 - a.janela) : 0;
        ns = min(a.sumid, lo);
        nvis = ns + q.i + 1 - lo;
    }
    const int x0 = min((long long)s * a.fatia, (long long)nvis), x1 = min(x0 + a.fatia, nvis), pag = 1 << a.L.lgpag;

    int qv[VB / 4];
    const int ld = (a.H + 2 * a.Hk) * HD, col = h * HD + c * VB;
#pragma unroll
    for (int k = 0; k < VB / 4; k++) qv[k] = reinterpret_cast<const int*>(a.qm + (long long)r * ld + col)[k];
    const int eq = a.qE[(long long)r * (ld >> a.lgblk) + (col >> a.lgblk)];
    constexpr float LOG2E = 1.4426950408889634f;
    const float esc = LOG2E / __builtin_sqrtf((float)HD), incl = a.incl ? a.incl[h] * LOG2E : 0.f;

    float m = -INFINITY, l = 0.f, o[VB];
#pragma unroll
    for (int d = 0; d < VB; d++) o[d] = 0.f;
    const long long dv = (long long)a.Hk * pag;                        // slots between a token's key and its value
    for (int base = x0 + w * KPW * U; base < x1; base += NW * KPW * U) {
        int j[U], p[U];
        bool vis[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int x = base + u * KPW + lane / LPK, xx = min(x, x1 - 1);
            vis[u] = x < x1;
            j[u] = xx < ns ? xx : xx - ns + lo;
            p[u] = a.L.tab[(long long)q.b * a.L.P + (j[u] >> a.L.lgpag)];
        }
        int kv[U][VB / 4], vv[U][VB / 4], ek[U], ev[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            if ((unsigned)p[u] >= (unsigned)a.L.npag) {
                if (vis[u] && c == 0) reporta(E_ARG, a.kid, (long long)q.b * a.L.P + (j[u] >> a.L.lgpag), p[u], j[u]);
                p[u] = 0;
                vis[u] = false;
            }
            const long long vaga = (long long)hk * pag + (j[u] & (pag - 1));
            const int8_t *km = a.cm + p[u] * a.pag_m + vaga * HD + c * VB, *ke = a.cE + p[u] * a.pag_e + vaga * G + g;
#pragma unroll
            for (int k = 0; k < VB / 4; k++) {
                kv[u][k] = reinterpret_cast<const int*>(km)[k];
                vv[u][k] = reinterpret_cast<const int*>(km + dv * HD)[k];
            }
            ek[u] = ke[0];
            ev[u] = ke[dv * G];
        }
        float t[U], mn = m;
#pragma unroll
        for (int u = 0; u < U; u++) {
            int d = 0;
#pragma unroll
            for (int k = 0; k < VB / 4; k++) d = __builtin_amdgcn_sdot4(qv[k], kv[u][k], d, false);
            t[u] = atc::soma_grupo<LPK>(__builtin_ldexpf((float)d, eq + ek[u])) * esc - incl * (float)(q.i - j[u]);
            t[u] = vis[u] ? t[u] : -INFINITY;
            mn = fmaxf(mn, t[u]);
        }
        const float ref = mn == -INFINITY ? 0.f : mn, al = __builtin_amdgcn_exp2f(m - ref);
        m = mn;
        l *= al;
#pragma unroll
        for (int d = 0; d < VB; d++) o[d] *= al;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const float e = __builtin_amdgcn_exp2f(t[u] - ref);
            l += e;
            const float pv = vis[u] ? __builtin_ldexpf(e, ev[u]) : 0.f;
#pragma unroll
            for (int d = 0; d < VB; d++) o[d] += pv * (float)(int8_t)(vv[u][d / 4] >> (8 * (d % 4)));
        }
    }

    // the wave's groups: a common maximum, then sums in which every step halves the values a lane still holds
    float M = m;
#pragma unroll
    for (int x = LPK; x < 64; x *= 2) M = fmaxf(M, __shfl_xor(M, x));
    const float es = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - M);
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
    constexpr int RESTO = VB / KPW > 1 ? VB / KPW : 1;                 // values a lane is left with
    __shared__ float so[NW][HD], sm[NW], sl[NW];
#pragma unroll
    for (int d = 0; d < RESTO; d++) so[w][c * VB + d0 + d] = o[d];     // lanes with the same values write the same
    if (lane == 0) { sm[w] = M; sl[w] = l; }
    __syncthreads();
    if (threadIdx.x >= HD) return;
    float MM = sm[0], LL = 0.f, oo = 0.f;
#pragma unroll
    for (int k = 1; k < NW; k++) MM = fmaxf(MM, sm[k]);
#pragma unroll
    for (int k = 0; k < NW; k++) {
        const float f = sm[k] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sm[k] - MM);
        LL += sl[k] * f;
        oo += so[k][threadIdx.x] * f;
    }
    const long long part = ((long long)r * a.H + h) * a.S + s;
    a.o[part * HD + threadIdx.x] = oo;
    if (threadIdx.x == 0) { a.ml[2 * part] = MM; a.ml[2 * part + 1] = LL; }
}

// fp32 values of a block (LPB lanes x NV) to int8 mantissas and an exponent, rounded once, half to even: E = binary
// exponent of the largest |v| - 7, one up where a mantissa passes 127; the products by 2^-E are exact. A block below
// 2^-126 is zero; one that holds an infinity or a NaN raises E_EXP and is zero.
template <int NV, int LPB>
__device__ __forceinline__ int quant_f32(const float (&v)[NV], int8_t (&q)[NV], int kid, long long idx0) {
    int bits = 0;
#pragma unroll
    for (int k = 0; k < NV; k++) bits = max(bits, __float_as_int(v[k]) & 0x7fffffff);
    bits = g_max<LPB>(bits);
    int E = (bits >> 23) - 133;
    float f = __builtin_ldexpf(1.f, -E);
    if (__builtin_rintf(__int_as_float(bits) * f) > 127.f) { E++; f *= 0.5f; }
    if (bits >= 0x7f800000) reporta(E_EXP, kid, idx0, E, bits);
    const bool zero = E < -126 || bits >= 0x7f800000;
#pragma unroll
    for (int k = 0; k < NV; k++) q[k] = zero ? 0 : (int8_t)(int)__builtin_rintf(v[k] * f);
    return zero ? E_ZERO : E;
}

// Joins the splits of a row and head, o = sum 2^(m_s - m) o_s / sum 2^(m_s - m) l_s (zeros for a row without visible
// tokens), 4 columns a thread, and writes the row as a block tensor (TIPO 0), bfloat16 (1) or fp32 (2).
template <int BLK, int TIPO>
__global__ void __launch_bounds__(256) k_atc_junta(const float* __restrict__ ml, const float* __restrict__ po, void* __restrict__ out,
                                                   int8_t* __restrict__ oE, int C, int hd, int S, int kid) {
    const int r = blockIdx.x, col = (blockIdx.y * 256 + threadIdx.x) * 4;
    if (col >= C) return;
    const long long part = ((long long)r * (C / hd) + col / hd) * S;
    float M = -INFINITY, L = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < S; s++) M = fmaxf(M, ml[2 * (part + s)]);
    for (int s = 0; s < S; s++) {
        const float m = ml[2 * (part + s)];
        if (m == -INFINITY) continue;
        const float f = __builtin_amdgcn_exp2f(m - M);
        L += f * ml[2 * (part + s) + 1];
        const float4 x = *reinterpret_cast<const float4*>(po + (part + s) * hd + col % hd);
        v[0] += f * x.x; v[1] += f * x.y; v[2] += f * x.z; v[3] += f * x.w;
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int k = 0; k < 4; k++) v[k] *= inv;
    const long long x = (long long)r * C + col;
    if constexpr (TIPO == 0) {
        int8_t q[4];
        const int E = quant_f32<4, BLK / 4>(v, q, kid, x);
        grava_i8<4, false>((int8_t*)out + x, q);
        if (col % BLK == 0) oE[x / BLK] = (int8_t)E;
    } else if constexpr (TIPO == 1) {
        typedef __bf16 b4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<b4*>((__bf16*)out + x) = b4{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
    } else {
        *reinterpret_cast<float4*>((float*)out + x) = make_float4(v[0], v[1], v[2], v[3]);
    }
}

// ---------------------------------------------------------------------------------------------- values
// A block or raw tensor as floats (the inverse of de_f32), each value rounded once: block values are exact in both types
// (8 bits), raw ones are scaled in double precision and rounded to fp32. 8 values a lane; bound by its bytes.
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
