"""The paged cache at its edges: scores beyond fp32, malformed sequences found by every kernel, many sequences, rows of no
sequence before and behind them, caches and rows past 2^31 and 2^32 bytes, captured calls, other streams, no rows at all,
and shapes drawn at random."""
import numpy as np
import pytest
import torch

import recipe as R
from backends import GPU, host
from geracao import Caso
from jatai_amd.registro import ErroJatai
from test_gpu_cache import _atende, _perto

pytestmark = pytest.mark.gpu

# (query heads of a kv head, new tokens): one row, up to 16 and more rows that share keys; short contexts and split ones
CAMINHOS = [(1, 1, 50), (1, 1, 3000), (4, 1, 50), (4, 1, 3000), (1, 20, 50), (2, 30, 3000)]


def _chama(g, caso, lote, saida, C=None, qkv=None, **kw):
    C = C or (g.dev(caso.m), g.dev(caso.E))
    qkv = qkv or (g.dev(caso.qm), g.dev(caso.qE))
    if not hasattr(caso, "incl_gpu"):
        caso.incl_gpu = g.dev(caso.incl())
    return g.ops.atencao_cache(qkv, C, caso.camadas - 1, lote, incl=caso.incl_gpu, saida=saida, **kw)


@pytest.mark.parametrize("Gq,n,c", CAMINHOS)
def test_notas_alem_de_fp32(Gq, n, c):
    """Scores of 2^130 and more: NaN in float outputs, an exponent event for a block output; the other sequences' rows stand."""
    caso = Caso(31, [c, c + 7, c + 1], [n, n, n], 2, 64, 32, Gq=Gq, pag=64)
    ref, tol = caso.atencao(caso.incl())
    ruins = slice(caso.ini[1], caso.ini[2])
    cols = caso.H * 64 // 32
    caso.qE[ruins, :cols] = np.where(caso.qE[ruins, :cols] == -127, -127, 70)
    caso.qm[ruins, :caso.H * 64] |= 1                       # no row of zeros, whose scores would all be 0
    caso.qE[ruins, :cols] = 70
    for p in caso.tabela[1]:
        if p >= 0:
            caso.E[p, 1, 0] = 60
            caso.m[p, 1, 0] |= 1
    print("atencao_cache", Gq, n, c, flush=True)
    g = GPU(32)
    y = _chama(g, caso, caso.lote(g.dev, g.O), torch.float32).double().cpu().numpy()
    g.reg.fim_passo()
    assert np.isnan(y[ruins]).all()
    boas = np.r_[0:caso.ini[1], caso.ini[2]:caso.M]
    assert (np.abs(y[boas] - ref[boas]) <= tol[boas] + np.abs(ref[boas]) * 2.0 ** -24).all()
    _chama(g, caso, caso.lote(g.dev, g.O), None)
    with pytest.raises(ErroJatai):
        g.reg.fim_passo()


def test_chaves_grandes_perguntas_pequenas():
    """Keys of 2^100 under queries of 2^-110: the scores are small, whatever the factors are."""
    for Gq, n, c in CAMINHOS:
        caso = Caso(32, [c, c + 5], [n, n], 2, 128, 32, Gq=Gq, pag=64)
        caso.qE = np.where(caso.qE == -127, -127, caso.qE - 104).astype(np.int8)
        for p in caso.tabela[caso.tabela >= 0]:
            caso.E[p, 1, 0] = np.where(caso.E[p, 1, 0] == -127, -127, np.clip(caso.E[p, 1, 0].astype(int) + 106, -126, 112)).astype(np.int8)
        _atende(caso)


@pytest.mark.parametrize("Gq,n,c", CAMINHOS)
@pytest.mark.parametrize("que", ["longa", "curta", "recua", "depois", "pagina", "negativa"])
def test_malformadas(Gq, n, c, que):
    """Whatever kernel runs: a malformed sequence is reported by the attention and by the write, the sequences before it keep their rows."""
    caso = Caso(33, [c, c + 9, c + 1], [n, n, n], 2, 64, 32, Gq=Gq, pag=64)
    ref, tol = caso.atencao(caso.incl())
    teto = c + 9
    if que == "longa": caso.comp[1] = teto + 1
    elif que == "curta": caso.comp[1] = n - 1
    elif que == "recua": caso.ini[2] = 0
    elif que == "depois": caso.ini[2:] = caso.M + 5
    elif que == "pagina": caso.tabela[1, (c + 8) // 64] = caso.m.shape[0]
    else: caso.tabela[1, (c + 8) // 64] = -1
    print("malformada", que, Gq, n, c, flush=True)
    g = GPU(32)
    lote = g.O.Lote(g.dev(caso.tabela), g.dev(np.array(caso.comp, np.int32)), g.dev(caso.ini), n, teto)
    C, qkv = (g.dev(caso.m), g.dev(caso.E)), (g.dev(caso.qm), g.dev(caso.qE))
    y = _chama(g, caso, lote, torch.float32, C, qkv)
    with pytest.raises(ErroJatai, match="invalid argument"):
        g.reg.fim_passo()
    g.reg.novo_passo(0)
    if que != "recua":                                      # rows that two sequences claim are nobody's
        y = y.double().cpu().numpy()[:n]
        assert (np.abs(y - ref[:n]) <= tol[:n] + np.abs(ref[:n]) * 2.0 ** -24).all()
    g.ops.cache_grava(qkv, C, 1, lote)
    with pytest.raises(ErroJatai, match="invalid argument"):
        g.reg.fim_passo()


@pytest.mark.parametrize("Gq,blk,hd", [(1, 32, 64), (1, 128, 4), (3, 32, 32)])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_muitas_sequencias(Gq, blk, hd, n):
    """150 sequences, some empty, some with nothing new, and rows of no sequence before the first and behind the last."""
    comp = [0 if b % 11 == 5 else 1 + (b * 37) % 90 for b in range(150)]
    novos = [0 if b % 7 == 3 else min(c, 1 + (b * 5) % n) for b, c in enumerate(comp)]
    Hk = 64 if hd == 4 else 4
    caso = Caso(34, comp, novos, Hk, hd, blk, Gq=Gq, sobra=9)
    caso.ini += 4
    for saida in (torch.float32, None):
        y = _atende(caso, saida)
        y = y[0] if saida is None else y
        assert not y[:4].any() and not y[-5:].any()
    g = GPU(blk)
    C = g.dev(caso.m), g.dev(caso.E)
    g.ops.cache_grava((g.dev(caso.qm), g.dev(caso.qE)), C, 1, caso.lote(g.dev, g.O))
    g.reg.fim_passo()
    m, E = caso.escrito()
    assert np.array_equal(host(C[0]), m) and np.array_equal(host(C[1]), E)


@pytest.mark.parametrize("hd,blk,pag", [(4, 128, 1024), (16, 32, 512), (64, 32, 1024), (128, 128, 256), (32, 128, 1024)])
def test_paginas_grandes(hd, blk, pag):
    Hk = max(2, 128 // hd) * (1 if blk == 32 else 2)
    for novos in ([1, 1, 1], [5, 1, 9], [1, 300, 40]):
        _atende(Caso(35, [pag - 1, pag + 300, 2 * pag + 1], novos, Hk, hd, blk, pag=pag), torch.bfloat16)


def test_cache_alem_de_4_gib():
    """Pages at byte offsets past 2^32: read, written, copied."""
    g = GPU(32)
    grande = None
    for Gq, n in ((1, 1), (4, 1), (1, 40)):
        caso = Caso(36, [1500, 70], [n, n], 2, 64, 32, Gq=Gq, pag=1024)
        k, paginas = caso.m.shape[0], 10000
        if grande is None:
            grande = tuple(torch.empty(paginas, *x.shape[1:], dtype=torch.int8, device="cuda") for x in (caso.m, caso.E))
            assert grande[0].numel() > 2**32
        antes = paginas - k
        for d, x in zip(grande, (caso.m, caso.E)):
            d[antes:] = g.dev(x)
        tab = np.where(caso.tabela >= 0, caso.tabela + antes, -1).astype(np.int32)
        lote = g.O.Lote(g.dev(tab), g.dev(np.array(caso.comp, np.int32)), g.dev(caso.ini), n, 1500)
        print("cache grande", Gq, n, flush=True)
        y = _chama(g, caso, lote, torch.float32, grande)
        ref, tol = caso.atencao(caso.incl())
        _perto(y, ref, tol, 32, torch.float32)
        g.ops.cache_grava((g.dev(caso.qm), g.dev(caso.qE)), grande, 1, lote)
        g.ops.cache_copia(grande, [(antes + x, 5 + x) for x in range(k)] + [(antes, antes - 1)])
        g.reg.fim_passo()
        for d, x in zip(grande, caso.escrito()):
            assert np.array_equal(host(d[antes:]), x) and np.array_equal(host(d[5:5 + k]), x) and np.array_equal(host(d[antes - 1]), x[0])


def test_linhas_alem_de_2_gib():
    """Rows whose bytes lie past 2^31, read and written; the rows before them belong to no sequence."""
    g = GPU(32)
    M = 90000
    for novos in ([1, 1], [2, 1]):
        caso = Caso(37, [90, 33], novos, 64, 128, 32)
        qkv = torch.zeros(M, caso.qm.shape[1], dtype=torch.int8, device="cuda"), torch.full((M, caso.qE.shape[1]), -127, dtype=torch.int8, device="cuda")
        assert qkv[0].numel() > 2**31
        for d, x in zip(qkv, (caso.qm, caso.qE)):
            d[-caso.M:] = g.dev(x)
        lote = g.O.Lote(g.dev(caso.tabela), g.dev(np.array(caso.comp, np.int32)), g.dev(caso.ini + M - caso.M), max(novos), 90)
        C = g.dev(caso.m), g.dev(caso.E)
        print("linhas", novos, flush=True)
        y = _chama(g, caso, lote, torch.bfloat16, C, qkv)
        g.ops.cache_grava(qkv, C, 1, lote)
        g.reg.fim_passo()
        ref, tol = caso.atencao(caso.incl())
        _perto(y[-caso.M:], ref, tol, 32, torch.bfloat16)
        assert not y[:-caso.M].any()
        assert all(np.array_equal(host(d), x) for d, x in zip(C, caso.escrito()))


def test_gravadas():
    """Two captured calls over one cache, replayed in turn while lengths and tables change and eager calls run between."""
    g = GPU(32)
    casos = [Caso(38 + k, [900 + 300 * k, 40, 70], [n] * 3, 2, 64, 32, Gq=Gq, pag=64) for k, (Gq, n) in enumerate(((1, 1), (4, 1), (1, 30)))]
    teto = 1600
    grafos = []
    for caso in casos:
        tab = np.full((3, teto // 64), -1, np.int32)
        tab[:, :caso.P] = caso.tabela
        lote = g.O.Lote(g.dev(tab), g.dev(np.array(caso.comp, np.int32)), g.dev(caso.ini), caso.novos[0], teto)
        C, qkv = (g.dev(caso.m), g.dev(caso.E)), (g.dev(caso.qm), g.dev(caso.qE))
        chama = lambda c=caso, l=lote, C=C, q=qkv: (g.ops.cache_grava(q, C, 1, l), _chama(g, c, l, None, C, q), _chama(g, c, l, torch.float32, C, q, janela=100))[1:]
        chama()
        torch.cuda.synchronize()
        grafo = torch.cuda.CUDAGraph()
        try:
            with torch.cuda.graph(grafo):
                g.ops.lib.jt_stream(torch.cuda.current_stream().cuda_stream)
                y = chama()
        finally:
            g.ops.lib.jt_stream(None)
        grafos.append((grafo, y, lote, chama, caso))
    for volta in range(3):
        for grafo, y, lote, _, caso in grafos:
            lote.comp.copy_(torch.tensor([caso.comp[0] - 64 * volta, caso.comp[1] - volta, caso.comp[2]], dtype=torch.int32))
            lote.tabela[0, :3] = lote.tabela[0, :3].roll(1)
        for grafo, *_ in grafos:
            grafo.replay()
        torch.cuda.synchronize()
        for grafo, y, lote, chama, caso in grafos:
            (m, E), f = chama()
            assert torch.equal(m, y[0][0]) and torch.equal(E, y[0][1]) and torch.equal(f, y[1]) and bool(torch.isfinite(f).all())
    g.reg.fim_passo()


def test_outra_corrente():
    """On a stream that the caller names, in order with its own work there."""
    g = GPU(32)
    caso = Caso(41, [2000, 300], [1, 1], 2, 64, 32, pag=64)
    C, qkv, lote = (g.dev(caso.m), g.dev(caso.E)), (g.dev(caso.qm), g.dev(caso.qE)), caso.lote(g.dev, g.O)
    certo = _chama(g, caso, lote, torch.float32, C, qkv)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        g.ops.lib.jt_stream(s.cuda_stream)
        try:
            x = torch.zeros_like(qkv[0])
            x.copy_(qkv[0])
            y = _chama(g, caso, lote, torch.float32, C, (x, qkv[1])) + 0
        finally:
            g.ops.lib.jt_stream(None)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, certo)
    g.reg.fim_passo()


def test_sem_linhas():
    g = GPU(32)
    caso = Caso(42, [20, 5], [0, 0], 2, 64, 32)
    C, lote = (g.dev(caso.m), g.dev(caso.E)), g.O.Lote(g.dev(caso.tabela), g.dev(np.array(caso.comp, np.int32)), g.dev(caso.ini), 0, 20)
    q = torch.zeros(0, 6 * 64, dtype=torch.int8, device="cuda"), torch.zeros(0, 12, dtype=torch.int8, device="cuda")
    for saida in (None, torch.bfloat16, torch.float32):
        y = _chama(g, caso, lote, saida, C, q)
        assert (y[0] if saida is None else y).shape == (0, 128)
        z = g.ops.valores(y) if saida is None else y
        assert z.shape == (0, 128)
    g.ops.cache_grava(q, C, 1, lote)
    g.reg.fim_passo()
    assert np.array_equal(host(C[0]), caso.m)


@pytest.mark.parametrize("semente", range(24))
def test_ao_acaso(semente):
    """Lengths, heads, pages, windows and outputs drawn at random."""
    u = lambda t, a, b: int(R.uniform_int(R.substream(100 + semente, t), (1,), a, b)[0])
    us = lambda t, n, a, b: R.uniform_int(R.substream(100 + semente, t), (n,), a, b).tolist()
    blk, hd = (32, 128)[u("blk", 0, 1)], (4, 16, 32, 64, 128)[u("hd", 0, 4)]
    Gq = (1, 1, 2, 3, 5, 8)[u("Gq", 0, 5)] if hd >= 32 else 1
    Hk = max(1, blk // hd) * u("Hk", 1, 2)
    pag, B, mais = 16 << u("pag", 0, 3), u("B", 1, 9), (1, 6, 130)[u("mais", 0, 2)]
    comp = us("comp", B, 0, 700)
    novos = [min(c, n) for c, n in zip(comp, us("novos", B, 0, mais))]
    janela = (0, 0, 1, 30, 200)[u("janela", 0, 4)]
    caso = Caso(200 + semente, comp, novos, Hk, hd, blk, Gq=Gq, pag=pag, sobra=u("sobra", 0, 3) + (sum(novos) == 0))
    saida = (None, torch.bfloat16, torch.float32)[u("saida", 0, 2)]
    if saida is None and caso.H * hd % blk:
        saida = torch.float32
    _atende(caso, saida, com_incl=u("incl", 0, 1) == 1, janela=janela, sumid=u("sumid", 0, 40))
