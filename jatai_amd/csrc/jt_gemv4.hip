// Products of a few rows with 4-bit weights (no reference counterpart): what a model's step for single tokens spends its time
// reading. A weight is q s 2^eb: q in [-7, 7] of 4 bits, one scale s (8 bits) 2^eb per row and block of BLK columns.
//
// Packed form of W [N, K]: tiles of 16 rows x 128 columns, 1 KB each in the order a wave's lanes read them. Byte 4 a + i of
// lane l's 16 bytes holds row l % 16's columns 32 a + 8 (l / 16) + i (low four bits) and + 4 more (high), two's complement;
// esc bf16 [N / 16][K / 128][16][128 / BLK] = s 2^(eb - R_j), exact, and R int16 [N] = the row's largest eb. Rows and columns
// that the last tiles lack are zeros.
//
// The sum is the block format's, integers rounded once per block at the row's and column's largest exponents:
//   acc_ij = sum_b rnd(p_ijb s_jb 2^(eb_jb - R_j) 2^(ea_ib - RA_i) 2^-g), half to even, exponent RA_i + R_j + g,
// p the exact dot product of a block, g = log2(BLK) - 4: |p s 2^-g| <= BLK 2^7 2^3 255 2^-g < 2^22, and K <= 256 BLK keeps
// |acc| below 2^30. Integer sums: any split of K gives the same bits.
#include "jt_comum.h"

namespace gv4 {
typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));
constexpr int CT = 2, COLS = 16 * CT;            // column tiles of a wave, and their columns

struct Args {
    const int8_t *x, *xE;
    const int4* w;
    const uint16_t* esc;
    const int16_t* R;
    const int8_t *res, *resE;
    void* y;
    void* yE;
    int M, N, K, modo, KS, CG, kid;              // modo: 0 block, 1 raw, 2 block + residual, 3 relu^2; KS waves along K, CG along N
};
constexpr int MAGICO = 0x4B400000;               // bits of 1.5 * 2^23: a float there is spaced by 1
}  // namespace gv4

// A wave takes CT tiles of 16 columns and every KS-th 128 columns of K; X's rows are the MFMA's other operand, row m in slot
// 4 (m % 4) + m / 4 of its 16, so that results of M <= 4 rows lie in NR = 1 of a lane's 4 registers (M <= 8: 2). The nibbles
// go to the MFMA as 16 q: the high ones by a mask, the low ones by a shift and a mask. Per result and block: the product as
// a float (exact), one multiplication for the scale (exact), one FMA onto 1.5 * 2^23 whose single rounding is the block's,
// and an integer add of its bits. The KS waves add their sums in LDS.
//   What bounds it: the weights' bytes, the rounding close behind (3.3 VALU operations per result and block; 7 us of VALU at
// 16 rows), and the launch. Every workgroup reads all of X from the L2: as whole lines, 16 bytes a lane, through the wave's own
// LDS. Read in the MFMA's layout (8 bytes of 16 rows a load, a quarter of each line) X was what bounded it: 16 x 8192 x 8192
// 16.3 us, 11.2 this way (3.4 TB/s of weights; 9.9 at 4 rows). 16 waves a workgroup, two steps of weights in flight; four, or 8 waves: the same.
// More than 16 rows hold more registers: two tiles of 16 and 8 waves there (64 rows of 8192 x 8192: 33 us).
template <int BLK, int NR, int MT>
__global__ void __launch_bounds__(MT > 1 ? 512 : 1024) k_gemv4(gv4::Args a) {
    using namespace gv4;
    constexpr int G4 = 128 / BLK, RT = 16 * MT, GUARDA = ilog2_c(BLK) - 4;
    extern __shared__ float lds[];
    const int nb = a.K / BLK, Kt = (a.K + 127) / 128, Nt = (a.N + 15) / 16, cols = COLS * a.CG;
    float* rs = lds;                                                  // [nb][MT][4: m % 4][4: m / 4]
    int* RA = reinterpret_cast<int*>(rs + nb * RT);                   // [RT]
    int* soma = RA + RT;                                              // [RT][cols]
    constexpr int XS = 144;                                           // bytes of an X row's 128 in a wave's own piece of LDS
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6, c = lane >> 4, n = lane & 15;
    const int ks = w % a.KS, cg = w / a.KS, m0 = blockIdx.y * RT;
    int8_t* xl = reinterpret_cast<int8_t*>(soma + RT * cols) + w * RT * XS;
    const int nt0 = (blockIdx.x * a.CG + cg) * CT;

    // the exponents of the wave's first row of X, then its first steps' bytes: waiting for the exponents leaves those in flight
    int ex[4];
    const int8_t* e0 = a.xE + (long long)min(m0 + w, a.M - 1) * nb;
#pragma unroll
    for (int k = 0; k < 4; k++) ex[k] = e0[min(lane + 64 * k, nb - 1)];
    constexpr int D = 2;                                              // steps whose weights are in flight
    int4 W[D][CT];
    uint2 S[D][CT];
    v4i X[MT][2];                                                     // X's bytes of the next step: 16 a lane, 8 lanes a row, whole lines
    unsigned linha[MT][2];
#pragma unroll
    for (int t = 0; t < MT; t++)
#pragma unroll
        for (int k = 0; k < 2; k++) linha[t][k] = (unsigned)(min(m0 + 16 * t + 8 * k + lane / 8, a.M - 1) - min(m0, a.M - 1)) * a.K;
    const int8_t* x0 = a.x + (long long)min(m0, a.M - 1) * a.K;
    auto carrega_w = [&](int z, int kt) {
#pragma unroll
        for (int t = 0; t < CT; t++) {
            const long long tile = (long long)min(nt0 + t, Nt - 1) * Kt + kt;
            W[z][t] = (a.w + tile * 64)[lane];
            const uint16_t* s = a.esc + tile * 16 * G4;
            if constexpr (G4 == 4) S[z][t] = reinterpret_cast<const uint2*>(s)[n];
            else S[z][t].x = s[n];
        }
    };
    auto carrega_x = [&](int kt) {
        const int k = 128 * kt + 16 * (lane % 8), o = k < a.K ? k : 0;                 // past K the weights are zeros
#pragma unroll
        for (int t = 0; t < MT; t++)
#pragma unroll
            for (int i = 0; i < 2; i++) X[t][i] = *reinterpret_cast<const v4i*>(x0 + linha[t][i] + o);
    };
    carrega_x(min(ks, Kt - 1));
#pragma unroll
    for (int z = 0; z < D; z++) carrega_w(z, min(ks + z * a.KS, Kt - 1));

    for (int m = w; m < RT; m += nw) {                                // exponents of X's rows, as scales of each block
        if (m > w) {
            const int8_t* e = a.xE + (long long)min(m0 + m, a.M - 1) * nb;
#pragma unroll
            for (int k = 0; k < 4; k++) ex[k] = e[min(lane + 64 * k, nb - 1)];
        }
        const int mx = g_max<64>(max(max(ex[0], ex[1]), max(ex[2], ex[3])));
        if (lane == 0) RA[m] = mx;
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (lane + 64 * k < nb) rs[(lane + 64 * k) * RT + (m & ~15) + 4 * (m % 4) + (m / 4) % 4] = __builtin_ldexpf(1.f, ex[k] - mx - GUARDA - 4);
    }
    for (int k = threadIdx.x; k < RT * cols; k += blockDim.x) soma[k] = 0;
    __syncthreads();

    int acc[CT][MT][NR] = {}, conta = 0;
    auto guarda_x = [&] {                                             // row m of 16 goes to slot 4 (m % 4) + m / 4
#pragma unroll
        for (int t = 0; t < MT; t++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int m = 8 * i + lane / 8;
                *reinterpret_cast<v4i*>(xl + (16 * t + 4 * (m % 4) + m / 4) * XS + 16 * (lane % 8)) = X[t][i];
            }
    };
    auto usa = [&](int z, int kt) {
        v4i p[CT][MT];
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int b = min((128 * kt + 32 * q) / BLK, nb - 1);     // past K the weights are zeros: 0 is added, without a branch
            long wq[CT];
#pragma unroll
            for (int t = 0; t < CT; t++) {
                const int x = q == 0 ? W[z][t].x : q == 1 ? W[z][t].y : q == 2 ? W[z][t].z : W[z][t].w;
                wq[t] = (long)(((unsigned long)(unsigned)(x & 0xF0F0F0F0) << 32) | (unsigned)((x << 4) & 0xF0F0F0F0));
            }
#pragma unroll
            for (int u = 0; u < MT; u++) {
                const long xq = __builtin_bit_cast(long, *reinterpret_cast<const v2i*>(xl + (16 * u + n) * XS + 32 * q + 8 * c));
#pragma unroll
                for (int t = 0; t < CT; t++) p[t][u] = __builtin_amdgcn_mfma_i32_16x16x32_i8(xq, wq[t], BLK == 32 || q == 0 ? v4i{0, 0, 0, 0} : p[t][u], 0, 0, 0);
                if (BLK == 128 && q < 3) continue;
                const v4i r = *reinterpret_cast<const v4i*>(rs + b * RT + 16 * u + 4 * c);
#pragma unroll
                for (int t = 0; t < CT; t++) {
                    const unsigned s = (q & 2) && BLK == 32 ? S[z][t].y : S[z][t].x;
                    const float sc = __int_as_float(BLK == 32 && (q & 1) ? s & 0xffff0000u : s << 16);
#pragma unroll
                    for (int k = 0; k < NR; k++) acc[t][u][k] += __float_as_int(__builtin_fmaf((float)p[t][u][k], sc * __int_as_float(r[k]), 12582912.f));
                    if constexpr (NR < 4) asm volatile("" ::"v"(p[t][u]));             // keeps the unread registers of a product from other products
                }
            }
        }
        conta += 128 / BLK;
    };
    for (int kt = ks; kt < Kt; kt += D * a.KS) {
#pragma unroll
        for (int z = 0; z < D; z++) {
            const int k = kt + z * a.KS;
            if (k < Kt) {
                guarda_x();
                carrega_x(min(k + a.KS, Kt - 1));
                usa(z, k);
                carrega_w(z, min(k + D * a.KS, Kt - 1));
            }
        }
    }
    if (ks < Kt) {
#pragma unroll
        for (int t = 0; t < CT; t++)
#pragma unroll
            for (int u = 0; u < MT; u++)
#pragma unroll
                for (int k = 0; k < NR; k++) {
                    const int m = 16 * u + c + 4 * k;
                    atomicAdd(&soma[m * cols + COLS * cg + 16 * t + n], acc[t][u][k] - (int)((unsigned)conta * (unsigned)MAGICO));
                }
    }
    __syncthreads();

    const int c0 = blockIdx.x * cols, linhas = min(RT, a.M - m0);
    if (a.modo == 1) {
        for (int k = threadIdx.x; k < linhas * cols; k += blockDim.x) {
            const int m = k / cols, j = c0 + k % cols;
            if (j < a.N) {
                const long long o = (long long)(m0 + m) * a.N + j;
                reinterpret_cast<int*>(a.y)[o] = soma[k];
                reinterpret_cast<int16_t*>(a.yE)[o] = (int16_t)(RA[m] + a.R[j] + GUARDA);
            }
        }
        return;
    }
    constexpr int LPB = BLK / 4;
    for (int k = threadIdx.x; k < linhas * cols / 4; k += blockDim.x) {
        const int m = 4 * k / cols, j = c0 + 4 * k % cols;
        if (j >= a.N) continue;                                       // N is whole blocks, so a group of lanes goes together
        const long long o = (long long)(m0 + m) * a.N + j;
        int v[4], e[4];
        int8_t q8[4];
#pragma unroll
        for (int i = 0; i < 4; i++) { v[i] = soma[4 * k + i]; e[i] = RA[m] + a.R[j + i] + GUARDA; }
        int E = quant8_d<4, LPB>(v, e, q8, a.kid, o);
        if (a.modo != 0) {
            int y[4];
            if (a.modo == 2) {                                        // as k_soma: aligned 21 bits below the larger exponent
                int x4[4];
                le_i8(a.res + o, x4);
                const int ex = a.resE[o / BLK], ec = max(E, ex) - 21;
                const Desl da(ec - ex), db(ec - E);
#pragma unroll
                for (int i = 0; i < 4; i++) v[i] = da(x4[i]) + db(q8[i]);
                E = quant8_u<4, LPB>(v, ec, y, a.kid, o);
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) { const int h = max((int)q8[i], 0); v[i] = h * h; }
                E = quant8_u<4, LPB>(v, 2 * E, y, a.kid, o);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) q8[i] = (int8_t)y[i];
        }
        grava_i8<4, false>((int8_t*)a.y + o, q8);
        if (j % BLK == 0) reinterpret_cast<int8_t*>(a.yE)[o / BLK] = (int8_t)E;
    }
}

// A block tensor W [N, K] to the packed form. Per block: a = its largest |mantissa|; the scale a / 7 as s 2^-k, s of 8 bits,
// nearest (a / 7 never lies halfway); q = m 2^k / s, half to even, exactly; |q| <= 7 since |m| <= a and s 2^-k is within
// 2^-8 of a / 7. One workgroup per 16 rows; run once per weight, so nothing is tuned.
template <int BLK>
__global__ void __launch_bounds__(256) k_para4(const int8_t* __restrict__ m, const int8_t* __restrict__ E, int8_t* __restrict__ w4,
                                               uint16_t* __restrict__ esc, int16_t* __restrict__ R, int N, int K) {
    constexpr int G4 = 128 / BLK;
    __shared__ int sk[16][256], Rl[16];                               // s | k << 8 | (eb + 1024) << 16; 0 for a block of zeros
    const int nb = K / BLK, Kt = (K + 127) / 128, r0 = blockIdx.x * 16;
    if (threadIdx.x < 16) Rl[threadIdx.x] = 0;
    __syncthreads();
    for (int x = threadIdx.x; x < 16 * nb; x += 256) {
        const int r = x / nb, b = x % nb;
        int a = 0, s = 0, k = 0, eb = 0;
        if (r0 + r < N) {
            const int8_t* p = m + (long long)(r0 + r) * K + b * BLK;
            for (int d = 0; d < BLK; d += 16) {
                int v[16];
                le_i8(p + d, v);
#pragma unroll
                for (int i = 0; i < 16; i++) a = max(a, abs(v[i]));
            }
        }
        if (a) {
            while ((a << k) < 896) k++;                               // a 2^k in [896, 1792): a 2^k / 7 in [128, 256)
            s = (2 * (a << k) + 7) / 14;
            if (s == 256) { s = 128; k--; }
            eb = E[(long long)(r0 + r) * nb + b] - k + 1024;
            atomicMax(&Rl[r], eb);
        }
        sk[r][b] = s | k << 8 | eb << 16;
    }
    __syncthreads();
    if (threadIdx.x < 16 && r0 + (int)threadIdx.x < N) R[r0 + threadIdx.x] = (int16_t)(Rl[threadIdx.x] ? Rl[threadIdx.x] - 1024 : E_ZERO);
    for (int x = threadIdx.x; x < Kt * 16 * G4; x += 256) {
        const int b = x / (16 * G4) * G4 + x % G4, r = x / G4 % 16, v = b < nb ? sk[r][b] : 0;
        const int d = (v >> 16) - Rl[r];                              // scales 2^100 below the row's largest round every product to 0
        esc[(long long)blockIdx.x * Kt * 16 * G4 + x] = v && d > -100 ? (uint16_t)(__float_as_uint(__builtin_ldexpf((float)(v & 255), d)) >> 16) : 0;
    }
    for (int x = threadIdx.x; x < Kt * 64; x += 256) {
        const int kt = x / 64, l = x % 64, r = l % 16;
        uint8_t y[16];
#pragma unroll
        for (int a = 0; a < 4; a++) {
            const int col = kt * 128 + 32 * a + 8 * (l / 16), v = r0 + r < N && col < K ? sk[r][col / BLK] : 0, s = v & 255, k = v >> 8 & 255;
            int q[8] = {};
            if (s) {
                le_i8(m + (long long)(r0 + r) * K + col, q);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int num = 2 * (abs(q[i]) << k) + s;
                    int t = num / (2 * s);
                    if (num == 2 * s * t && (t & 1)) t--;             // a tie goes to the even one
                    q[i] = q[i] < 0 ? -t : t;
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) y[4 * a + i] = (uint8_t)((q[i] & 15) | (q[4 + i] & 15) << 4);
        }
        int4 z;
        z.x = y[0] | y[1] << 8 | y[2] << 16 | y[3] << 24; z.y = y[4] | y[5] << 8 | y[6] << 16 | y[7] << 24;
        z.z = y[8] | y[9] << 8 | y[10] << 16 | y[11] << 24; z.w = y[12] | y[13] << 8 | y[14] << 16 | y[15] << 24;
        reinterpret_cast<int4*>(w4)[((long long)blockIdx.x * Kt + kt) * 64 + l] = z;
    }
}
