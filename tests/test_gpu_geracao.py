"""Generation: every operator of a run checked on the inputs that the run gave it (the training operators bit for bit against
the CPU oracle, the new ones against their 64-bit forms), and the run's own promises: the captured step gives the eager
one's bits at every replay, forks and compactions change nothing, and errors name their step."""
import numpy as np
import pytest
import torch

import recipe as R
from backends import LOGS, host
from geracao import vale
from test_gpu_cache import _perto
from test_gpu_gemv4 import desempacota, produto

pytestmark = pytest.mark.gpu

MODELOS = {"cab64": (256, 256, 4, 512, 2, 32), "cab4": (256, 256, 64, 512, 2, 128), "cab32": (256, 128, 4, 256, 1, 32)}


def _modelo(nome, r16=False, embrulho=None):
    from jatai_amd import ops as O
    from jatai_amd.modelo import Modelo
    from jatai_amd.registro import Registro
    V, D, H, FF, L, blk = MODELOS[nome]
    O.BLK = blk
    reg = Registro(LOGS, "geracao", eco=False)
    ops = O.OpsHip(reg)
    if embrulho:
        ops = embrulho(ops, blk)
    return Modelo(V, D, H, FF, L, 3, "cuda", ops, reg, r16=r16)


def _texto(semente, n, V=256):
    return R.tokens(semente, n, V).tolist()


class Conferido:
    """OpsHip with every call of a generation checked on its own inputs."""

    def __init__(self, ops, blk):
        from oracle.ops_oracle import OpsOraculo
        self.ops, self.reg, self.lib, self.blk, self.spec, self.vistas = ops, ops.reg, ops.lib, blk, OpsOraculo(blk), []

    def __getattr__(self, nome):
        if nome in ("inclinacoes", "para4"):
            return getattr(self.ops, nome)
        if nome not in ("embed", "rms", "gemm", "gemm_soma", "gemm_relu2", "para16", "para8", "soma16", "valores", "cache_grava", "cache_copia", "atencao_cache",
                        "gemv4", "gemv4_soma", "gemv4_relu2"):
            raise AttributeError(nome)
        f = getattr(self.ops, nome)

        def chama(*a, **k):
            antes = [t.clone() for t in a[1]] if nome == "cache_grava" else None
            y = f(*a, **k)
            self.vistas.append(nome)
            getattr(self, "_" + nome, self._spec)(nome, y, a, k) if nome != "cache_grava" else self._grava(y, a, antes)
            return y
        return chama

    @staticmethod
    def _iguais(nome, y, z):
        if isinstance(y, tuple):
            assert len(y) == len(z), nome
            for p, q in zip(y, z):
                Conferido._iguais(nome, p, q)
        else:
            assert np.array_equal(host(y), np.asarray(z)), nome

    def _spec(self, nome, y, a, k):
        self._iguais(nome, y, getattr(self.spec, nome)(*a, **k))

    def _embed(self, nome, y, a, k):
        self._iguais(nome, y, self.spec.embed(a[0], a[1].cpu()))

    def _valores(self, nome, y, a, k):
        m, E = host(a[0][0]), host(a[0][1])
        assert np.array_equal(host(y), (np.ldexp(m.astype(np.float64), E) if m.dtype == np.int32 else vale(m, E, self.blk)).astype(np.float32))

    def _gemv4(self, nome, y, a, k):
        X, P = a[:2]
        x, xE, N = host(X[0]), host(X[1]), P[2].numel()
        acc, e = produto(x, xE, *desempacota(P, N, x.shape[1], self.blk), self.blk)
        cru = torch.from_numpy(acc.astype(np.int32)), torch.from_numpy(e.astype(np.int16))
        h = cru if k.get("cru") else self.spec.quant(cru)
        self._iguais(nome, y, self.spec.soma(a[2], h) if nome == "gemv4_soma" else self.spec.relu2(h) if nome == "gemv4_relu2" else h)
    _gemv4_soma = _gemv4_relu2 = _gemv4

    def _linhas(self, qkv, lote):
        """(row, sequence, position) of every row that has a sequence."""
        comp = host(lote.comp)
        if lote.ini is None:
            return [(b, b, c - 1) for b, c in enumerate(comp) if c > 0]
        ini = host(lote.ini)
        return [(ini[b] + t, b, comp[b] - (ini[b + 1] - ini[b]) + t) for b in range(len(comp)) for t in range(ini[b + 1] - ini[b])]

    def _grava(self, C, a, antes):
        qkv, _, camada, lote = a
        (m, E), (pages, L, _, Hk, pag, hd) = [host(t).copy() for t in antes], antes[0].shape
        qm, qE, tab, gs = host(qkv[0]), host(qkv[1]), host(lote.tabela), min(hd, self.blk)
        H = qm.shape[1] // hd - 2 * Hk
        col = np.arange((H + 2 * Hk) * hd // gs) * gs // self.blk
        for r, b, j in self._linhas(qkv, lote):
            p = tab[b, j // pag]
            m[p, camada, :, :, j % pag] = qm[r].reshape(-1, hd)[H:].reshape(2, Hk, hd)
            E[p, camada, :, :, j % pag] = qE[r, col].reshape(H + 2 * Hk, -1)[H:].reshape(2, Hk, -1)
        assert np.array_equal(host(C[0]), m) and np.array_equal(host(C[1]), E)

    def _cache_copia(self, nome, y, a, k):
        pass                                                         # what it moved is read by the attention that follows

    def _atencao_cache(self, nome, y, a, k):
        qkv, C, camada, lote, incl, janela, sumid = a
        Hk, pag, hd = C[0].shape[3:]
        gs, H, incl, tab = min(hd, self.blk), incl.numel(), host(incl), host(lote.tabela)
        q = vale(host(qkv[0]), host(qkv[1]), self.blk)[:, :H * hd].reshape(-1, H, hd)
        kv = vale(host(C[0][:, camada]), host(C[1][:, camada]), gs)      # [pages, 2, Hk, pag, hd]
        ref, tol = np.zeros(q.shape), np.zeros(q.shape)
        for r, b, i in self._linhas(qkv, lote):
            j = np.arange(i + 1)
            j = j[(j > i - janela) | (j < sumid)] if janela else j
            p = tab[b, j // pag]
            assert (p >= 0).all()
            x = kv[p, :, :, j % pag]                                   # [n, 2, Hk, hd]
            for h in range(H):
                kk, v, bias = x[:, 0, h * Hk // H], x[:, 1, h * Hk // H], incl[h] * (i - j)
                u = kk @ q[r, h] / np.sqrt(hd) - bias
                w = np.exp(u - u.max())
                w /= w.sum()
                rel = w * (8 * (np.abs(kk) @ np.abs(q[r, h]) / np.sqrt(hd) + np.abs(bias)) + 8)
                ref[r, h] = w @ v                                     # the bound of geracao.Caso.atencao
                tol[r, h] = 2.0 ** -24 * (rel @ np.abs(v) + rel.sum() * np.abs(ref[r, h]) + (len(j) + 32) * (w @ np.abs(v) + np.abs(ref[r, h]))) \
                    + 2.0 ** -126 * (np.abs(v).sum(0) + len(j) + 1)
        _perto(y, ref.reshape(len(q), -1), tol.reshape(len(q), -1), self.blk, None)


def _gerador(m, **kw):
    from jatai_amd.geracao import Gerador
    kw = dict(dict(seqs=3, max_tokens=160, pagina=16), **kw)
    return Gerador(m, **kw)


@pytest.mark.parametrize("nome,r16,kw", [("cab64", False, {}), ("cab64", True, {}), ("cab64", False, dict(bits=4)), ("cab64", True, dict(bits=4)),
                                         ("cab64", False, dict(janela=20, sumidouros=3)), ("cab4", False, {}), ("cab4", False, dict(bits=4, janela=33)),
                                         ("cab32", False, dict(bits=4))])
def test_cada_operador_de_uma_geracao(nome, r16, kw):
    """Ragged prompts, a continuation of one of them, then a step of each (the step's eager form, whose bits the captured one has)."""
    m = _modelo(nome, r16, Conferido)
    g = _gerador(m, **kw)
    y = g.le({2: _texto(1, 41), 0: _texto(2, 3)})
    assert y.shape == (2, m.V) and y.dtype == torch.float32
    g.le({0: _texto(3, 17), 1: _texto(4, 1)})
    vistas = set(m.ops.vistas)
    assert {"embed", "rms", "cache_grava", "atencao_cache", "valores"} <= vistas and ("gemv4_relu2" in vistas) == (kw.get("bits") == 4)
    g.cache.reserva({0: 1, 2: 1})
    g.cache.envia()
    from jatai_amd import ops as O
    comp = torch.tensor([g.cache.n[0], 0, g.cache.n[2]], dtype=torch.int32).cuda()
    tok = torch.zeros(g.linhas, dtype=torch.int32, device="cuda")
    tok[:3] = torch.tensor([7, 0, 9], dtype=torch.int32)
    g._camadas(tok, O.Lote(g.cache.tabela, comp, None, 1, 160))
    m.reg.fim_passo()


@pytest.mark.parametrize("nome,kw", [("cab64", {}), ("cab64", dict(bits=4)), ("cab64", dict(janela=24, sumidouros=2)), ("cab4", {})])
def test_passo_gravado_igual_ao_eager(nome, kw):
    """Replays of the captured step, with other work, synchronizations and changes of the live sequences in between, against
    the same step op by op on a second cache: logits, choices and caches bit for bit."""
    from jatai_amd import ops as O
    m = _modelo(nome)
    a, b = _gerador(m, **kw), _gerador(m, **kw)
    for g in (a, b):
        g.le({0: _texto(1, 30), 1: _texto(2, 14), 2: _texto(3, 47)})
    tok = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    for k in range(24):
        vivas = [0, 1, 2] if k < 8 else [0, 2] if k < 14 else [1] if k < 16 else [0, 1, 2]
        logits, escolha = a.passo(vivas, tok)
        b.cache.reserva({s: 1 for s in vivas})
        b.cache.envia()
        comp = torch.tensor([b.cache.n[s] if s in vivas else 0 for s in range(3)], dtype=torch.int32).cuda()
        t = torch.zeros(b.linhas, dtype=torch.int32, device="cuda")
        t[:3] = tok
        y = b._camadas(t, O.Lote(b.cache.tabela, comp, None, 1, 160))[:3]
        b._esquece()
        assert torch.equal(logits, y)
        assert escolha.tolist() == [int(min(torch.nonzero(r == r.max())).item()) for r in y.cpu()]
        if k % 5 == 0:
            torch.cuda.synchronize()
            _ = torch.randn(512, 512, device="cuda").sum().item()
        if k == 10:                                                  # a continuation between replays
            for g in (a, b):
                g.le({1: _texto(9, 5)})
        if k == 12:
            assert a.cache.compacta() == b.cache.compacta()
        tok = escolha.clone()
    a.confere()
    m.reg.fim_passo()
    assert a.cache.n == b.cache.n and torch.equal(a.cache.C[0], b.cache.C[0]) and torch.equal(a.cache.C[1], b.cache.C[1])


def test_bifurca_compacta_e_libera():
    """Two forks of a prompt that go on differently equal two sequences that read everything themselves, with pages freed and
    moved in between."""
    m = _modelo("cab64")
    a, b = _gerador(m, seqs=4, paginas=14), _gerador(m, seqs=4, paginas=40)
    p = _texto(5, 37)
    a.le({0: _texto(6, 60)})
    a.le({1: p})
    a.cache.bifurca(1, 2)
    a.cache.libera(0)
    assert a.cache.livres == 14 - 3
    ya = a.le({1: [5], 2: [6]})                                        # both write into the shared last page: one copy
    assert a.cache.livres == 14 - 4 and a.cache.compacta() > 0
    b.le({1: p, 2: p})
    yb = b.le({1: [5], 2: [6]})
    assert torch.equal(ya, yb)
    tok = torch.tensor([0, 8, 9, 0], dtype=torch.int32, device="cuda")
    for _ in range(20):
        za, zb = a.passo([1, 2], tok)[0], b.passo([1, 2], tok)[0]
        assert torch.equal(za[1:3], zb[1:3])
        a.cache.compacta()
        tok = a.escolha.clone()
    a.confere()
    b.confere()


def test_gera():
    m = _modelo("cab64")
    g = _gerador(m)
    textos = [_texto(7, 20), _texto(8, 1)]
    saida = g.gera(textos, 12)
    assert [len(t) for t in saida] == [12, 12] and all(0 <= x < m.V for t in saida for x in t)
    assert saida == g.gera(textos, 12) and g.cache.n == [0] * 3 and g.cache.livres == 30
    fixa = g.gera(textos, 5, escolhe=lambda y: torch.full((len(y),), 65, device="cuda"))
    assert fixa == [[65] * 5] * 2 and g.gera([], 4) == [] and g.gera(textos, 0) == [[], []]


def test_recusas_do_gerador():
    from jatai_amd.registro import ErroJatai
    m = _modelo("cab64")
    g = _gerador(m, paginas=5)
    tok = torch.zeros(3, dtype=torch.int32, device="cuda")
    for f in (lambda: g.le({}), lambda: g.le({0: []}), lambda: g.le({0: [256]}), lambda: g.le({0: [-1]}), lambda: g.le({3: [1]}), lambda: g.le({0: [1] * 161}),
              lambda: g.le({0: [1] * 81}), lambda: g.passo([0, 0], tok), lambda: g.passo([0], tok[:2]), lambda: g.passo([3], tok), lambda: g.gera([[1]] * 4, 2),
              lambda: g.gera([[1] * 70, [1] * 70], 2), lambda: _gerador(m, bits=5)):
        with pytest.raises(ErroJatai):
            f()
        assert g.cache.n == [0] * 3 and g.cache.livres == 5
    g.le({0: [1, 2, 3]})


def test_evento_num_passo_gravado():
    """A page outside the cache, planted in the device table, is reported by the captured step with its operation and scope."""
    from jatai_amd.registro import ErroJatai
    m = _modelo("cab64")
    g = _gerador(m)
    g.le({0: _texto(1, 20)})
    tok = torch.zeros(3, dtype=torch.int32, device="cuda")
    g.passo([0], tok)
    g.confere()
    g.cache.tabela[0, 0] = 10**6
    g.passo([0], tok)
    with pytest.raises(ErroJatai, match="atencao_cache") as e:
        g.confere()
    assert "passo / camada 0 / atencao" in str(e.value) and "valor    : 1000000" in str(e.value)


def test_evento_de_um_entre_dois_geradores():
    """The device has one event record: another generator's steps and prompts do not clear what one has yet to read."""
    from jatai_amd.registro import ErroJatai
    tok = torch.zeros(3, dtype=torch.int32, device="cuda")
    for depois in ("passo", "le"):
        a, b = _gerador(_modelo("cab64")), _gerador(_modelo("cab64"))
        for g in (a, b):
            g.le({0: _texto(1, 20)})
            g.passo([0], tok)
            g.confere()
        a.cache.tabela[0, 0] = 10**6
        a.passo([0], tok)
        if depois == "passo":
            b.passo([0], tok)
            with pytest.raises(ErroJatai, match="invalid argument"):
                a.confere()
            with pytest.raises(ErroJatai):
                b.confere()
        else:
            with pytest.raises(ErroJatai, match="invalid argument"):
                b.le({1: _texto(2, 5)})
        b.le({2: _texto(3, 5)})                                        # the record is cleared once everyone has read it
        b.passo([0], tok)
        b.confere()


def test_desalinhados():
    """Contiguous tensors that do not begin at 16 bytes are refused; nothing is written."""
    from backends import GPU
    from jatai_amd.registro import ErroJatai
    g = GPU(32)
    torto = lambda *f: torch.zeros(int(torch.Size(f).numel()) + 8, dtype=torch.int8, device="cuda")[3:-5].view(f)
    reto = lambda *f: torch.zeros(f, dtype=torch.int8, device="cuda")
    i32 = lambda *f: torch.zeros(f, dtype=torch.int32, device="cuda")
    lote = g.O.Lote(i32(2, 1), i32(2), None, 1, 16)
    qkv, C = (lambda m: (m, reto(4, 12))), (lambda m: (m, reto(6, 1, 2, 2, 16, 2)))
    X, P = (lambda m: (m, reto(3, 4))), g.ops.para4((reto(32, 128), reto(32, 4)))
    for f in (lambda: g.ops.cache_grava(qkv(torto(4, 384)), C(reto(6, 1, 2, 2, 16, 64)), 0, lote), lambda: g.ops.cache_grava(qkv(reto(4, 384)), C(torto(6, 1, 2, 2, 16, 64)), 0, lote),
              lambda: g.ops.atencao_cache(qkv(torto(4, 384)), C(reto(6, 1, 2, 2, 16, 64)), 0, lote), lambda: g.ops.cache_copia(C(torto(6, 1, 2, 2, 16, 64)), [(0, 1)]),
              lambda: g.ops.gemv4(X(torto(3, 128)), P), lambda: g.ops.para4((torto(32, 128), reto(32, 4))), lambda: g.ops.valores(X(torto(3, 128)))):
        with pytest.raises(ErroJatai, match="refused the launch"):
            f()
    g.reg.fim_passo()
