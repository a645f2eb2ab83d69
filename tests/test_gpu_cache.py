"""The paged cache on the GPU: its page operators bit for bit, and attention over it against the 64-bit form, at every
head width and block size, lengths from one token on, ragged batches, shared heads, windows, and pages that end anywhere."""
import numpy as np
import pytest
import torch

from backends import GPU, host
from geracao import Caso, vale

pytestmark = pytest.mark.gpu

FORMAS = [(4, 32, 16), (4, 128, 64), (16, 32, 16), (16, 128, 32), (32, 32, 64), (32, 128, 16), (64, 32, 64), (64, 128, 16), (128, 32, 32), (128, 128, 128)]


def _hk(hd, blk, Gq=1):
    """Heads whose row of queries, keys and values, and whose output, are whole blocks."""
    return max(2, 128 // hd) * (1 if blk == 32 else 2)


def _perto(y, ref, tol, blk, saida):
    if saida is None:
        m, E = host(y[0]), host(y[1])
        v = vale(m, E, blk)
        passo = np.ldexp(0.5, np.repeat(E.astype(np.int32), blk, axis=1))
        zero = E == -127
        assert (np.abs(m.reshape(E.shape[0], -1, blk)).max(2)[~zero] >= 63).all() and not m.reshape(E.shape[0], -1, blk)[zero].any()
        lim = np.where(np.repeat(zero, blk, axis=1), 2.0 ** -119, passo) + tol
    else:
        v = y.double().cpu().numpy()
        lim = tol + np.abs(ref) * torch.finfo(saida).eps / 2
    d = np.abs(v - ref) - lim
    assert np.isfinite(v).all() and (d <= 0).all(), (float(d.max()), np.unravel_index(d.argmax(), d.shape), v.flat[d.argmax()], ref.flat[d.argmax()])


def _atende(caso, saida=torch.float32, com_incl=True, janela=0, sumid=0, com_ini=True):
    g = GPU(caso.blk)
    incl = caso.incl() if com_incl else None
    print(f"atencao_cache hd {caso.hd} blk {caso.blk} pag {caso.pag} comp {caso.comp} novos {caso.novos} Hk {caso.Hk} Gq {caso.Gq} janela {janela} {sumid} {saida}", flush=True)
    C = g.dev(caso.m), g.dev(caso.E)
    y = g.ops.atencao_cache((g.dev(caso.qm), g.dev(caso.qE)), C, caso.camadas - 1, caso.lote(g.dev, g.O, com_ini), incl=g.dev(incl) if com_incl else None,
                            janela=janela, sumidouros=sumid, saida=saida)
    g.reg.fim_passo()
    ref, tol = caso.atencao(incl, janela, sumid)
    _perto(y, ref, tol, caso.blk, saida)
    assert np.array_equal(host(C[0]), caso.m) and np.array_equal(host(C[1]), caso.E)
    return y


@pytest.mark.parametrize("hd,blk,pag", FORMAS)
@pytest.mark.parametrize("saida", [None, torch.bfloat16, torch.float32])
def test_token_novo(hd, blk, pag, saida):
    """One new token per sequence, from a sequence of a single token to several pages; with and without row starts."""
    caso = Caso(1, [1, 2, 15, 16, 17, 63, 64, 65, 130, 700], [1] * 10, _hk(hd, blk), hd, blk, pag=pag)
    a = _atende(caso, saida)
    b = _atende(caso, saida, com_ini=False)
    for x, y in zip(a if saida is None else (a,), b if saida is None else (b,)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("hd,blk,pag", FORMAS)
def test_linhas_de_varios_tamanhos(hd, blk, pag):
    """Ragged rows: prompts (every token new), continuations, sequences with nothing new or nothing at all, and rows behind
    the last sequence, which come out as zeros."""
    caso = Caso(2, [70, 0, 33, 200, 1, 90], [70, 0, 1, 5, 1, 0], _hk(hd, blk), hd, blk, pag=pag, sobra=3)
    for saida in (torch.float32, None):
        y = _atende(caso, saida)
        y = y[0] if saida is None else y
        assert not y[-3:].any() and bool(y[:-3].any())


@pytest.mark.parametrize("hd,blk,pag", [f for f in FORMAS if f[0] >= 16])
@pytest.mark.parametrize("Gq", [2, 3, 8])
def test_cabecas_partilhadas(hd, blk, pag, Gq):
    """Query heads that share keys and values, a new token and several."""
    caso = Caso(3, [40, 129, 5], [1, 1, 1], _hk(hd, blk), hd, blk, Gq=Gq, pag=pag)
    _atende(caso)
    caso = Caso(4, [40, 129, 5], [7, 30, 5], _hk(hd, blk), hd, blk, Gq=Gq, pag=pag)
    _atende(caso, torch.bfloat16)


@pytest.mark.parametrize("hd,blk,pag", [(64, 32, 16), (64, 32, 64), (4, 128, 16), (128, 128, 32)])
@pytest.mark.parametrize("janela,sumid", [(1, 0), (1, 1), (7, 4), (64, 0), (65, 70), (300, 1), (5000, 9)])
def test_janela(hd, blk, pag, janela, sumid):
    """Windows and first tokens, for new tokens and for rows whose windows differ; the pages in between are gone (-1)."""
    comp = [1, 20, 400, 333]
    for novos in ([1, 1, 1, 1], [1, 20, 40, 3]):
        solta = [(b, p) for b, c in enumerate(comp) for p in range(c // pag) if p * pag >= sumid and (p + 1) * pag <= c - novos[b] + 1 - janela]
        _atende(Caso(5, comp, novos, _hk(hd, blk), hd, blk, pag=pag, solta=solta), torch.float32, janela=janela, sumid=sumid)


def test_sem_inclinacao_e_longo():
    """No position bias over a context of several splits; a bias that leaves only the nearest tokens."""
    caso = Caso(6, [5000, 4097], [1, 1], 2, 64, 32, pag=64)
    _atende(caso, com_incl=False)
    _atende(caso, com_incl=True)
    _atende(Caso(6, [3000], [70], 2, 64, 32, pag=64), com_incl=False)


def test_expoentes_extremos():
    """Values whose exponents lie far apart (blocks from 2^-60 to 2^6 of one another) and blocks of zeros."""
    for e0 in (-40, 3):
        caso = Caso(7, [50, 77], [1, 4], 2, 64, 32, e0=e0, zera=0.4)
        caso.E[:, :, 1] = np.where(caso.E[:, :, 1] > 20, 20, caso.E[:, :, 1]) if e0 > 0 else caso.E[:, :, 1]
        if e0 > 0:                                    # scores up to a few thousand: the softmax is one-hot
            caso.qE = np.where(caso.qE == -127, -127, caso.qE - 6).astype(np.int8)
        _atende(caso)


@pytest.mark.parametrize("hd,blk,pag", FORMAS)
@pytest.mark.parametrize("Gq", [1, 3])
def test_grava(hd, blk, pag, Gq):
    caso = Caso(8, [70, 0, 33, 200, 1, 90], [70, 0, 1, 5, 1, 0], _hk(hd, blk), hd, blk, Gq=Gq, pag=pag, sobra=2)
    um = Caso(9, [70, 3, 33], [1, 1, 1], _hk(hd, blk), hd, blk, Gq=Gq, pag=pag)
    for c, com_ini in ((caso, True), (um, True), (um, False)):
        g = GPU(blk)
        C = g.dev(c.m), g.dev(c.E)
        Z = g.ops.cache_grava((g.dev(c.qm), g.dev(c.qE)), C, c.camadas - 1, c.lote(g.dev, g.O, com_ini))
        g.reg.fim_passo()
        m, E = c.escrito()
        assert Z[0] is C[0] and np.array_equal(host(C[0]), m) and np.array_equal(host(C[1]), E)


@pytest.mark.parametrize("hd,blk,pag,camadas", [(4, 128, 16, 1), (64, 32, 64, 3), (128, 32, 16, 2)])
def test_copia(hd, blk, pag, camadas):
    caso = Caso(10, [pag * 600], [1], 2 if hd > 4 else 64, hd, blk, pag=pag, camadas=camadas)
    for pares in ([], [(3, 5)], [(0, 601), (0, 2), (7, 600)], [(k, 301 + k) for k in range(300)]):
        g = GPU(blk)
        C = g.dev(caso.m), g.dev(caso.E)
        g.ops.cache_copia(C, pares)
        g.reg.fim_passo()
        m, E = caso.m.copy(), caso.E.copy()
        for d, p in pares:
            m[p], E[p] = caso.m[d], caso.E[d]
        assert np.array_equal(host(C[0]), m) and np.array_equal(host(C[1]), E)


@pytest.mark.parametrize("blk", [32, 128])
def test_valores(blk):
    import recipe as R
    g = GPU(blk)
    m, E = R.bloco(11, 5, 3 * 128, blk, espalha=110, e0=0, zera=0.2)
    for tipo in (torch.float32, torch.bfloat16):
        y = g.ops.valores((g.dev(m), g.dev(E)), tipo)
        assert y.dtype == tipo and np.array_equal(y.double().cpu().numpy(), vale(m, E, blk))
    acc, e = R.cru(12, 7, 33)
    e[0, :4] = [-180, -170, 90, 0]
    acc[0, :4] = [3, 2**29 + 1, 2**29 - 1, 0]
    y = g.ops.valores((g.dev(acc), g.dev(e)))
    g.reg.fim_passo()
    assert np.array_equal(host(y), np.ldexp(acc.astype(np.float64), e).astype(np.float32))


def _mal(muda, **kw):
    """A call on malformed device data: reported, nothing read out of bounds, the other sequences' rows as they should be."""
    from jatai_amd.registro import ErroJatai
    caso = Caso(13, [40, 50, 60], [1, 2, 1], 2, 64, 32, pag=16)
    ref, tol = caso.atencao(caso.incl())
    muda(caso)
    g = GPU(32)
    C, qkv = (g.dev(caso.m), g.dev(caso.E)), (g.dev(caso.qm), g.dev(caso.qE))
    lote = g.O.Lote(g.dev(caso.tabela), g.dev(np.array(caso.comp, np.int32)), g.dev(caso.ini), kw.get("novos", 2), kw.get("teto", 60))
    y = g.ops.atencao_cache(qkv, C, 1, lote, incl=g.dev(caso.incl()), saida=torch.float32)
    with pytest.raises(ErroJatai, match="invalid argument"):
        g.reg.fim_passo()
    g.reg.novo_passo(0)
    d = np.abs(y.double().cpu().numpy() - ref) - tol - np.abs(ref) * 2.0 ** -24
    g.ops.cache_grava(qkv, C, 1, lote)
    with pytest.raises(ErroJatai, match="invalid argument"):
        g.reg.fim_passo()
    return y, d


def test_dados_malformados():
    def comp(c): c.comp[1] = 61
    def curto(c): c.comp[1] = 1
    def pagina(c): c.tabela[1, 3] = c.m.shape[0]
    def negativa(c): c.tabela[1, 3] = -1
    def ini(c): c.ini[2] = 7
    for muda in (comp, curto, pagina, negativa):
        y, d = _mal(muda)
        assert (d[[0, 3]] <= 0).all() and bool(torch.isfinite(y).all())
        if muda in (comp, curto):
            assert not y[1:3].any()
    y, d = _mal(ini)
    assert (d[0] <= 0).all() and bool(torch.isfinite(y).all())
    y, d = _mal(lambda c: None, novos=1)
    assert (d[[0, 3]] <= 0).all() and not y[1:3].any()
