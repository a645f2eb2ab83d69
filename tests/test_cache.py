"""The cache's bookkeeping without a GPU: every step of a random run of reservations, forks, releases, forgotten windows and
compactions against a model that keeps each sequence's tokens in a list; refusals; the C entry points' host checks."""
import ctypes
import random

import pytest
import torch

from jatai_amd import ops as O
from jatai_amd.cache import CacheKV
from jatai_amd.registro import ErroJatai, Registro


class OpsFalso:
    """cache_copia on a list of page contents."""

    def __init__(self, tmp, paginas):
        self.reg, self.conteudo = Registro(str(tmp), "cache", eco=False), [None] * paginas

    def cache_copia(self, C, pares):
        para = [p for _, p in pares]
        assert len(set(para)) == len(para) and not set(para) & {d for d, _ in pares}
        for d, p in pares:
            self.conteudo[p] = dict(self.conteudo[d])


def _cache(tmp, paginas=20, seqs=5, max_tokens=64, pagina=16):
    ops = OpsFalso(tmp, paginas)
    return ops, CacheKV(ops, 1, 2, 16, paginas, seqs, max_tokens, pagina, dev="cpu")


def _confere(ops, c, modelo, esquecidas):
    for s, toks in enumerate(modelo):
        assert c.n[s] == len(toks) and len(c.paginas[s]) == -(-len(toks) // c.pagina)
        for i, p in enumerate(c.paginas[s]):
            if (s, i) in esquecidas:
                assert p == -1
            else:
                assert {k: v for k, v in ops.conteudo[p].items() if k < len(toks) - i * c.pagina} == dict(enumerate(toks[i * c.pagina:(i + 1) * c.pagina]))
    usos = [0] * len(c.usos)
    for ps in c.paginas:
        for p in ps:
            if p >= 0:
                usos[p] += 1
    assert usos == c.usos and sorted(c._livres) == [p for p, u in enumerate(usos) if u == 0]
    c.envia()
    assert c.comp.tolist() == c.n and [[p for p in ps] for ps in c.paginas] == [t[:len(ps)] for t, ps in zip(c.tabela.tolist(), c.paginas)]
    assert all(x == -1 for t, ps in zip(c.tabela.tolist(), c.paginas) for x in t[len(ps):])


@pytest.mark.parametrize("semente", range(8))
def test_ao_acaso(tmp_path, semente):
    rng = random.Random(semente)
    ops, c = _cache(tmp_path)
    modelo, esquecidas, proximo = [[] for _ in range(5)], set(), 0
    recusas = 0
    for _ in range(400):
        acao = rng.choice(["reserva"] * 5 + ["bifurca", "libera", "esquece", "compacta"])
        if acao == "reserva":
            novos = {s: rng.choice([0, 1, 1, 2, 17]) for s in rng.sample(range(5), rng.randint(1, 5))}
            antes = (list(c.n), [list(p) for p in c.paginas], list(c.usos), sorted(c._livres))
            try:
                c.reserva(novos)
            except ErroJatai:
                recusas += 1
                assert antes == (c.n, c.paginas, c.usos, sorted(c._livres))
                continue
            for s, k in novos.items():                               # the model's kernel: each new token into its slot
                for _ in range(k):
                    j, proximo = len(modelo[s]), proximo + 1
                    p = c.paginas[s][j // 16]
                    assert c.usos[p] == 1
                    if ops.conteudo[p] is None or j % 16 == 0:
                        ops.conteudo[p] = {}
                    ops.conteudo[p][j % 16] = proximo
                    modelo[s].append(proximo)
        elif acao == "bifurca":
            de, para = rng.sample(range(5), 2)
            if modelo[para] or c.paginas[para]:
                with pytest.raises(ErroJatai):
                    c.bifurca(de, para)
                continue
            c.bifurca(de, para)
            modelo[para] = list(modelo[de])
            esquecidas |= {(para, i) for s, i in esquecidas if s == de}
        elif acao == "libera":
            s = rng.randrange(5)
            c.libera(s)
            modelo[s] = []
            esquecidas = {x for x in esquecidas if x[0] != s}
        elif acao == "esquece":
            s, janela, sumid = rng.randrange(5), rng.choice([1, 5, 16, 17, 40]), rng.choice([0, 1, 16, 20])
            c.esquece(s, janela, sumid)
            n = len(modelo[s])
            for i in range(len(c.paginas[s])):
                vistos = [j for j in range(16 * i, 16 * i + 16) if j > n - janela or j < sumid]
                if not vistos:
                    esquecidas.add((s, i))
        else:
            usadas = sum(u > 0 for u in c.usos)
            fora = sum(u > 0 for u in c.usos[usadas:])
            assert c.compacta() == fora and all(u > 0 for u in c.usos[:usadas]) and not any(c.usos[usadas:])
        _confere(ops, c, modelo, esquecidas)
    assert recusas


def test_recusas(tmp_path):
    ops, c = _cache(tmp_path)
    for chamada in (lambda: c.reserva({5: 1}), lambda: c.reserva({0: -1}), lambda: c.reserva({0: 65}), lambda: c.reserva({0: 64, 1: 64, 2: 64, 3: 64, 4: 64, "a": 1}),
                    lambda: c.bifurca(1, 1), lambda: c.bifurca(0, 9), lambda: c.libera(-1), lambda: c.esquece(0, 0), lambda: c.esquece(0, 4, -1)):
        with pytest.raises(ErroJatai):
            chamada()
        assert c.livres == 20 and c.n == [0] * 5
    c.reserva({0: 64, 1: 64, 2: 64, 3: 64, 4: 64})
    assert c.livres == 0
    c.esquece(0, 1)
    assert c.paginas[0] == [-1] * 4 and c.livres == 4          # a whole window of one token: the next token sees only itself


def test_guardas_c_sem_gpu():
    """Malformed calls return hipErrorInvalidValue before anything is launched (there is no GPU to launch on here, and none
    of the addresses is read)."""
    lib = O.carrega_lib()
    assert lib.jt_bloco(32) == 0
    p, n = ctypes.c_void_p(1 << 20), ctypes.c_void_p(0)
    par = lambda *v: ctypes.cast((ctypes.c_int * len(v))(*v), ctypes.c_void_p)
    copia = dict(cm=p, cE=p, npag=10, camadas=1, Hk=2, hd=64, pag=16, pares=par(0, 1), n=1, kid=0)
    assert lib.jt_cache_copia(*{**copia, "n": 0}.values()) == 0
    for muda in (dict(cm=n), dict(cE=ctypes.c_void_p((1 << 20) + 8)), dict(npag=0), dict(hd=48), dict(pag=24), dict(pag=8), dict(n=-1), dict(pares=n),
                 dict(pares=par(0, 10)), dict(pares=par(-1, 3)), dict(pares=par(0, 0)), dict(pares=par(0, 1, 2, 1), n=2), dict(pares=par(0, 1, 1, 2), n=2)):
        assert lib.jt_cache_copia(*{**copia, **muda}.values()) == 1, muda
    lote = dict(tab=p, comp=p, ini=p, M=4, B=2, P=4, novos=2, teto=64)
    grava = dict(qm=p, qE=p, cm=p, cE=p, npag=10, camadas=2, camada=1, Hk=2, hd=64, pag=16, **lote, H=2, kid=0)
    assert lib.jt_cache_grava(*{**grava, "M": 0}.values()) == 0
    ruins = (dict(qm=n), dict(qE=n), dict(cm=n), dict(cE=n), dict(npag=0), dict(camada=2), dict(camada=-1), dict(Hk=0), dict(hd=8), dict(pag=48), dict(tab=n),
             dict(comp=n), dict(M=-1), dict(B=0), dict(P=0), dict(novos=-1), dict(teto=2**30), dict(teto=-1), dict(qm=ctypes.c_void_p((1 << 20) + 4)))
    for muda in ruins + (dict(H=-1), dict(H=70000)):
        assert lib.jt_cache_grava(*{**grava, **muda}.values()) == 1, muda
    nws = lib.jt_atencao_cache_ws_bytes(4, 2, 4, 2, 64, 2, 8192, 0, 0, 0)
    at = dict(qm=p, qE=p, cm=p, cE=p, npag=10, camadas=2, camada=1, Hk=2, hd=64, pag=16, tab=p, comp=p, ini=p, incl=n, out=p, outE=p, M=4, B=2, P=512, novos=2,
              teto=8192, H=4, janela=0, sumid=0, tipo=0, ws=p, nws=ctypes.c_longlong(nws), kid=0)
    assert nws > 0 and lib.jt_atencao_cache(*{**at, "M": 0}.values()) == 0
    for muda in ruins + (dict(teto=8193), dict(H=3), dict(H=0), dict(out=n), dict(outE=n), dict(janela=-1), dict(sumid=-1), dict(tipo=3), dict(tipo=-1), dict(ws=n),
                         dict(nws=ctypes.c_longlong(nws - 1)), dict(ws=ctypes.c_void_p((1 << 20) + 4))):
        assert lib.jt_atencao_cache(*{**at, **muda}.values()) == 1, muda
    val = dict(m=p, E=p, out=p, n=ctypes.c_longlong(64), cru=0, tipo=1, kid=0)
    for muda in (dict(m=n), dict(E=n), dict(out=n), dict(n=ctypes.c_longlong(-1)), dict(n=ctypes.c_longlong(33)), dict(cru=2), dict(cru=1), dict(tipo=0)):
        assert lib.jt_valores(*{**val, **muda}.values()) == 1, muda
    para = dict(m=p, E=p, w=p, esc=p, R=p, N=5, K=128, kid=0)
    for muda in (dict(m=n), dict(w=n), dict(N=0), dict(K=0), dict(K=48), dict(K=32 * 257), dict(esc=ctypes.c_void_p(4))):
        assert lib.jt_para4(*{**para, **muda}.values()) == 1, muda
    gv = dict(x=p, xE=p, w=p, esc=p, R=p, res=n, resE=n, y=p, yE=p, M=3, N=64, K=128, modo=0, kid=0)
    assert lib.jt_gemv4(*{**gv, "M": 0}.values()) == 0
    for muda in (dict(x=n), dict(xE=n), dict(w=n), dict(esc=n), dict(R=n), dict(y=n), dict(yE=n), dict(M=-1), dict(N=0), dict(N=33), dict(K=48), dict(K=32 * 257),
                 dict(modo=2), dict(modo=4), dict(modo=-1), dict(x=ctypes.c_void_p((1 << 20) + 8))):
        assert lib.jt_gemv4(*{**gv, **muda}.values()) == 1, muda
    lib.jt_bloco(O.BLK)


def test_guardas_python_sem_gpu(tmp_path, monkeypatch):
    """The operators' own checks, on tensors that report a GPU; nothing is launched."""
    class NaGpu(torch.Tensor):
        is_cuda = property(lambda self: True)
        dispositivo = 0

        def get_device(self):
            return self.dispositivo

    def z(*forma, tipo=torch.int8):
        return torch.zeros(*forma, dtype=tipo).as_subclass(NaGpu)

    def outra(t):
        t.dispositivo = 1
        return t
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(O, "BLK", 32)
    ops = object.__new__(O.OpsHip)
    ops.reg, ops._blk = Registro(str(tmp_path), "g", eco=False), 32

    def proibe(*a, **k):
        raise AssertionError("launched")
    ops._lanca = proibe
    i32 = torch.int32
    C, qkv = (z(6, 2, 2, 2, 16, 64), z(6, 2, 2, 2, 16, 2)), (z(4, 384), z(4, 12))
    lote = O.Lote(z(2, 3, tipo=i32), z(2, tipo=i32), z(3, tipo=i32), 4, 48)
    at = lambda q=qkv, c=C, camada=0, l=lote, **k: ops.atencao_cache(q, c, camada, l, **k)
    gr = lambda q=qkv, c=C, camada=0, l=lote: ops.cache_grava(q, c, camada, l)
    for f in (at, gr):
        for kw in (dict(q=(z(4, 384), z(4, 11))), dict(q=(z(4, 320), z(4, 10))), dict(q=(z(4, 256), z(4, 8))), dict(camada=2), dict(camada=-1),
                   dict(c=(z(6, 2, 2, 2, 16, 48), z(6, 2, 2, 2, 16, 1))), dict(c=(z(6, 2, 2, 2, 24, 64), z(6, 2, 2, 2, 24, 2))), dict(c=(C[0], z(6, 2, 2, 2, 16, 1))),
                   dict(c=(z(6, 2, 1, 2, 16, 64), z(6, 2, 1, 2, 16, 2))), dict(c=(z(0, 2, 2, 2, 16, 64), z(0, 2, 2, 2, 16, 2))),
                   dict(c=(z(6, 2, 2, 2, 64, 16).transpose(4, 5), C[1])), dict(c=(outra(z(6, 2, 2, 2, 16, 64)), C[1])), dict(q=(outra(z(4, 384)), z(4, 12))),
                   dict(l=lote._replace(tabela=z(2, 3))), dict(l=lote._replace(tabela=z(3, 3, tipo=i32))), dict(l=lote._replace(comp=z(2, 1, tipo=i32))),
                   dict(l=lote._replace(ini=z(2, tipo=i32))), dict(l=lote._replace(teto=49)), dict(l=lote._replace(teto=-1)), dict(l=lote._replace(novos=-1)),
                   dict(l=lote._replace(tabela=z(3, 2, tipo=i32).t())), dict(l=lote._replace(comp=outra(z(2, tipo=i32)))),
                   dict(l=O.Lote(z(5, 3, tipo=i32), z(5, tipo=i32), None, 1, 48))):
            with pytest.raises(ErroJatai):
                f(**kw)
    for kw in (dict(janela=-1), dict(sumidouros=-1), dict(saida=torch.float16), dict(incl=z(2)), dict(incl=z(3, tipo=torch.float32))):
        with pytest.raises(ErroJatai):
            at(**kw)
    for pares in ([(0, 6)], [(-1, 2)], [(0, 0)], [(0, 1), (2, 1)], [(0, 1), (1, 2)], [(0,), (1, 2)]):
        with pytest.raises(ErroJatai):
            ops.cache_copia(C, pares)
    with pytest.raises(ErroJatai):
        ops.valores((z(4, 5, tipo=i32), z(4, 5, tipo=torch.int16)), torch.bfloat16)
    with pytest.raises(ErroJatai):
        ops.valores(qkv, torch.float16)
    with pytest.raises(ErroJatai):
        ops.para4((z(4, 32 * 257), z(4, 257)))
    W = (z(3, 2, 64, 16, tipo=torch.uint8), z(3, 2, 16, 4, tipo=torch.bfloat16), z(48, tipo=torch.int16))
    X = (z(5, 160), z(5, 5))
    for w, x, modo in ((W, X, 0), (W, (z(5, 128), z(5, 4)), 1), ((W[0], W[1][:, :, :, :1], W[2]), X, 1), ((W[0], W[1], z(49, tipo=torch.int16)), X, 1),
                       ((z(3, 2, 64, 16), W[1], W[2]), X, 1), ((outra(z(3, 2, 64, 16, tipo=torch.uint8)), W[1], W[2]), X, 1)):
        with pytest.raises(ErroJatai):
            ops._gemv4("gemv4", modo, x, w)
    W64 = (z(4, 2, 64, 16, tipo=torch.uint8), z(4, 2, 16, 4, tipo=torch.bfloat16), z(64, tipo=torch.int16))
    with pytest.raises(ErroJatai):
        ops.gemv4_soma(X, W64, (z(5, 96), z(5, 3)))


def test_recusas_de_construcao(tmp_path):
    ops = OpsFalso(tmp_path, 4)
    for a in ((0, 2, 16, 4, 2, 32, 16), (1, 0, 16, 4, 2, 32, 16), (1, 2, 8, 4, 2, 32, 16), (1, 2, 16, 0, 2, 32, 16), (1, 2, 16, 4, 0, 32, 16), (1, 2, 16, 4, 2, 0, 16),
              (1, 2, 16, 4, 2, 32, 24), (1, 2, 16, 4, 2, 32, 8), (1, 2, 16, 4, 2, 32, 2048)):
        with pytest.raises(ErroJatai, match="CacheKV"):
            CacheKV(ops, *a, dev="cpu")


def test_outro_dispositivo(tmp_path, monkeypatch):
    """Operands that lie on different GPUs, or on another than the current one, are refused before anything is launched."""
    class NaGpu(torch.Tensor):
        is_cuda = property(lambda self: True)
        dispositivo = 0

        def get_device(self):
            return self.dispositivo

    def z(*forma, tipo=torch.int8, d=0):
        t = torch.zeros(*forma, dtype=tipo).as_subclass(NaGpu)
        t.dispositivo = d
        return t
    atual = [0]
    monkeypatch.setattr(torch.cuda, "current_device", lambda: atual[0])
    monkeypatch.setattr(O, "BLK", 32)
    ops = object.__new__(O.OpsHip)
    ops.reg, ops._blk, lancados = Registro(str(tmp_path), "g", eco=False), 32, []
    ops._lanca = lambda op, *a, **k: lancados.append(op)
    bf, i16, i32 = torch.bfloat16, torch.int16, torch.int32
    usos = [(lambda m, E: ops.valores((m, E)), [(z, (4, 64)), (z, (4, 2))]),
            (lambda a, e: ops.valores((a, e)), [(lambda *f, d=0: z(*f, tipo=i32, d=d), (4, 64)), (lambda *f, d=0: z(*f, tipo=i16, d=d), (4, 64))]),
            (lambda m, E: ops.para4((m, E)), [(z, (32, 128)), (z, (32, 4))]),
            (lambda x, xE, w, s, r, m, E: ops.gemv4_soma((x, xE), (w, s, r), (m, E)),
             [(z, (3, 128)), (z, (3, 4)), (lambda *f, d=0: z(*f, tipo=torch.uint8, d=d), (2, 1, 64, 16)), (lambda *f, d=0: z(*f, tipo=bf, d=d), (2, 1, 16, 4)),
              (lambda *f, d=0: z(*f, tipo=i16, d=d), (32,)), (z, (3, 32)), (z, (3, 1))]),
            (lambda m, E, cm, cE, t, c: ops.cache_grava((m, E), (cm, cE), 0, O.Lote(t, c, None, 1, 16)),
             [(z, (4, 384)), (z, (4, 12)), (z, (6, 1, 2, 2, 16, 64)), (z, (6, 1, 2, 2, 16, 2)), (lambda *f, d=0: z(*f, tipo=i32, d=d), (2, 1)),
              (lambda *f, d=0: z(*f, tipo=i32, d=d), (2,))])]
    for f, partes in usos:
        lancados.clear()
        f(*(g(*forma) for g, forma in partes))
        assert len(lancados) == 1
        for k in range(len(partes)):
            with pytest.raises(ErroJatai):
                f(*(g(*forma, d=int(i == k)) for i, (g, forma) in enumerate(partes)))
        atual[0] = 1
        with pytest.raises(ErroJatai):
            f(*(g(*forma) for g, forma in partes))
        atual[0] = 0
        assert len(lancados) == 1
