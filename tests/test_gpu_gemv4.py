"""Products with 4-bit weights on the GPU, bit for bit: the packing against exact rationals, the product against 64-bit
integers, its fused forms against the ops they fuse, at every number of rows per tile, odd sizes and both block sizes."""
import numpy as np
import pytest
import torch

import recipe as R
from backends import GPU, host

pytestmark = pytest.mark.gpu


def desempacota(P, N, K, blk):
    """(q [N, K], scales [N, K / blk] as float64, R) of the packed form."""
    w, esc, r = host(P[0]), P[1].double().cpu().numpy(), host(P[2])
    Nt, Kt = w.shape[:2]
    t = w.reshape(Nt, Kt, 4, 16, 4, 4)                               # tile, tile, l // 16, l % 16, a, i
    t = np.stack([t & 15, t >> 4], axis=-1).astype(np.int64)
    t = np.where(t > 7, t - 16, t).transpose(0, 3, 1, 4, 2, 6, 5).reshape(Nt * 16, Kt * 128)
    e = esc.transpose(0, 2, 1, 3).reshape(Nt * 16, -1)
    assert not t[N:].any() and not t[:, K:].any() and not e[N:].any() and not e[:, K // blk:].any()
    return t[:N, :K], e[:N, :K // blk], r


def produto(xm, xE, q, esc, r, blk):
    """acc, e of the definition: per block the exact dot product times the 8-bit scale, shifted with half to even."""
    M, K = xm.shape
    N, nb, g = len(q), K // blk, {32: 1, 128: 3}[blk]
    RA = xE.astype(np.int64).max(1)
    f, t = np.frexp(esc)
    s8, t = (f * 256).astype(np.int64), 8 - t.astype(np.int64)
    acc = np.zeros((M, N), np.int64)
    for b in range(nb):
        p = (xm[:, b * blk:(b + 1) * blk].astype(np.int64) @ q[:, b * blk:(b + 1) * blk].T) * s8[:, b]
        sh = np.minimum((RA - xE[:, b])[:, None] + t[:, b] + g, 62)
        piso, um = p >> sh, np.int64(1)
        resto = p - (piso << sh)
        meio = um << (sh - 1)
        acc += piso + ((resto > meio) | ((resto == meio) & (piso & 1 == 1)))
    return acc, RA[:, None] + r + g


def _pesos(semente, N, K, blk):
    m, E = R.bloco(semente, N, K, blk, espalha=5, e0=-9, zera=0.1)
    m[0], E[0] = 0, -127                                             # a row of zeros
    if N > 3:
        m[1, :blk], m[2, :blk], m[3, :blk] = 1, -127, 127            # blocks of one value
        E[1, 0] = -126
        m[3, 0] = -128
    return m, E


@pytest.mark.parametrize("blk", [32, 128])
@pytest.mark.parametrize("N,K", [(16, 128), (1, 128), (50, 384), (128, 512), (33, 256 * 32)])
def test_para4(blk, N, K):
    m, E = _pesos(1, N, K, blk)
    g = GPU(blk)
    P = g.ops.para4((g.dev(m), g.dev(E)))
    g.reg.fim_passo()
    q, esc, r = desempacota(P, N, K, blk)
    mb = np.abs(m.astype(np.int64)).reshape(N, K // blk, blk).max(2)
    for j in range(N):
        vivos = [b for b in range(K // blk) if mb[j, b]]
        eb = {}
        for b in vivos:
            a, k = int(mb[j, b]), 0
            while (a << k) < 896:
                k += 1
            s = (2 * (a << k) + 7) // 14                             # nearest: a 2^k / 7 has no ties
            s, k = (128, k - 1) if s == 256 else (s, k)
            eb[b] = (int(E[j, b]) - k, s, k)
        Rj = max((v[0] for v in eb.values()), default=-127)
        assert r[j] == Rj
        for b in range(K // blk):
            e, s, k = eb.get(b, (0, 0, 0))
            assert esc[j, b] == (s * 2.0 ** (e - Rj) if s and e - Rj > -100 else 0)
            x = m[j, b * blk:(b + 1) * blk].astype(np.int64)
            if not s:
                assert not q[j, b * blk:(b + 1) * blk].any()
                continue
            num = np.abs(x) << k
            t, resto = num // s, num % s
            t += (2 * resto > s) | ((2 * resto == s) & (t & 1 == 1))
            assert t.max() == 7 and np.array_equal(q[j, b * blk:(b + 1) * blk], np.sign(x) * t)


@pytest.mark.parametrize("blk", [32, 128])
@pytest.mark.parametrize("M", [1, 3, 4, 5, 8, 9, 16, 17, 32, 33, 64, 65, 130])
@pytest.mark.parametrize("N,K", [(128, 128), (1, 384), (50, 640), (300, 128 * 20)])
def test_gemv4_cru(blk, M, N, K):
    m, E = _pesos(2, N, K, blk)
    xm, xE = R.bloco(R.substream(3, f"{M}"), M, K, blk, espalha=6, e0=-4, zera=0.1)
    if M > 4:
        xm[1], xE[1] = 0, -127
    g = GPU(blk)
    P = g.ops.para4((g.dev(m), g.dev(E)))
    acc, e = g.ops.gemv4((g.dev(xm), g.dev(xE)), P, cru=True)
    g.reg.fim_passo()
    a, ee = produto(xm, xE, *desempacota(P, N, K, blk), blk)
    assert np.array_equal(host(acc), a) and np.array_equal(host(e), ee)


@pytest.mark.parametrize("blk,K", [(32, 32), (32, 96), (32, 32 * 256), (128, 128 * 256), (32, 32 * 133)])
def test_gemv4_comprimentos(blk, K):
    """K from one block to the largest, at the largest mantissas (sums just below 2^30), all of one sign."""
    M, N = 2, 32
    g = GPU(blk)
    for extremo in (False, True):
        m, E = _pesos(4, N, K, blk)
        xm, xE = R.bloco(5, M, K, blk, espalha=6, e0=-4)
        P = g.ops.para4((g.dev(m), g.dev(E)))
        if extremo:                                                  # every weight -8 and scale 255, every activation -128
            P = (torch.full_like(P[0], 0x88), torch.full_like(P[1], 255), torch.zeros_like(P[2]))
            if K % 128:
                P[1][:, -1, :, K // blk % (128 // blk):] = 0
                P[0][:, -1].view(-1, 64, 4, 4)[:, :, K % 128 // 32:] = 0
            xm, xE = np.full_like(xm, -128), np.zeros_like(xE)
        acc, e = g.ops.gemv4((g.dev(xm), g.dev(xE)), P, cru=True)
        a, ee = produto(xm, xE, *desempacota(P, N, K, blk), blk)
        assert np.abs(a).max() < 2 ** 30 and np.array_equal(host(acc), a) and np.array_equal(host(e), ee)
    g.reg.fim_passo()


@pytest.mark.parametrize("blk", [32, 128])
@pytest.mark.parametrize("M", [1, 7, 16, 40])
@pytest.mark.parametrize("N,K", [(128, 256), (384, 512), (896, 1664)])
def test_gemv4_fundido(blk, M, N, K):
    """Block output, residual add and relu^2 equal quant, soma and relu2 of the raw product; the raw output is unchanged."""
    m, E = _pesos(6, N, K, blk)
    xm, xE = R.bloco(7, M, K, blk, espalha=6, e0=-4, zera=0.1)
    rm, rE = R.bloco(8, M, N, blk, espalha=12, e0=-6, zera=0.1)
    g = GPU(blk)
    P = g.ops.para4((g.dev(m), g.dev(E)))
    X, res = (g.dev(xm), g.dev(xE)), (g.dev(rm), g.dev(rE))
    h = g.ops.quant(g.ops.gemv4(X, P, cru=True))
    for y, z in ((g.ops.gemv4(X, P), h), (g.ops.gemv4_soma(X, P, res), g.ops.soma(res, h)), (g.ops.gemv4_relu2(X, P), g.ops.relu2(h))):
        assert torch.equal(y[0], z[0]) and torch.equal(y[1], z[1])
    g.reg.fim_passo()


def test_pesos_alem_de_2_gib():
    """The last rows of weights whose packed bytes pass 2^31 (and whose mantissas pass 2^32): packed and multiplied as by themselves."""
    N, K, blk, n = 270000, 16384, 128, 64
    m, E = _pesos(9, n, K, blk)
    xm, xE = R.bloco(10, 3, K, blk, espalha=6, e0=-4)
    g = GPU(blk)
    W = torch.zeros(N, K, dtype=torch.int8, device="cuda"), torch.full((N, K // blk), -127, dtype=torch.int8, device="cuda")
    for d, x in zip(W, (m, E)):
        d[-n:] = g.dev(x)
    P, p = g.ops.para4(W), g.ops.para4((g.dev(m), g.dev(E)))
    assert P[0].numel() > 2**31 and all(torch.equal(a[-b.shape[0]:], b) for a, b in zip(P, p))
    X = g.dev(xm), g.dev(xE)
    (acc, e), (a, ee) = g.ops.gemv4(X, P, cru=True), g.ops.gemv4(X, p, cru=True)
    g.reg.fim_passo()
    assert torch.equal(acc[:, -n:], a) and torch.equal(e[:, -n:], ee) and not acc[:, :-n].any() and bool(a.any())


def test_gemv4_sem_linhas_gravado_e_noutra_corrente():
    blk, N, K = 32, 256, 640
    g = GPU(blk)
    P = g.ops.para4(tuple(map(g.dev, _pesos(11, N, K, blk))))
    z = g.ops.gemv4((torch.zeros(0, K, dtype=torch.int8, device="cuda"), torch.zeros(0, K // blk, dtype=torch.int8, device="cuda")), P)
    assert z[0].shape == (0, N) and z[1].shape == (0, N // blk)
    entradas = [tuple(map(g.dev, R.bloco(R.substream(12, f"{k}"), 5, K, blk, espalha=6, e0=-4))) for k in range(3)]
    res = tuple(map(g.dev, R.bloco(13, 5, N, blk, e0=-6)))
    certas = [g.ops.valores(g.ops.gemv4_soma(X, P, res)) for X in entradas]
    X = tuple(t.clone() for t in entradas[0])
    torch.cuda.synchronize()
    grafo = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(grafo):
            g.ops.lib.jt_stream(torch.cuda.current_stream().cuda_stream)
            y = g.ops.valores(g.ops.gemv4_soma(X, P, res))
    finally:
        g.ops.lib.jt_stream(None)
    for novo, certa in list(zip(entradas, certas)) * 2:
        for d, o in zip(X, novo):
            d.copy_(o)
        grafo.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, certa) and torch.equal(g.ops.valores(g.ops.gemv4_soma(novo, P, res)), certa)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        g.ops.lib.jt_stream(s.cuda_stream)
        try:
            y = g.ops.valores(g.ops.gemv4_soma(tuple(t.clone() for t in entradas[1]), P, res)) + 0
        finally:
            g.ops.lib.jt_stream(None)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, certas[1])
    g.reg.fim_passo()
