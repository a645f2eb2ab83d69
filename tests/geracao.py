"""Inputs and the plain 64-bit form of the generation operators, for their tests: a cache of random pages with garbage in
the slots no token holds, ragged sequences, and attention over them with the error that fp32 arithmetic may leave."""
import numpy as np

import recipe as R


def vale(m, E, n):
    """Values of mantissas whose last axis takes one exponent per n columns, float64."""
    return m.astype(np.float64) * np.ldexp(1.0, np.repeat(E.astype(np.int32), n, axis=-1))


class Caso:
    """comp, novos: tokens and new tokens of each sequence; Hk heads of width hd, H = Hk Gq query heads. The cache holds
    every sequence's tokens, the new ones' keys and values too; pages are handed out shuffled. `sobra`: rows behind the
    last sequence. `solta`: page runs (b, p) whose table entry is -1."""

    def __init__(self, semente, comp, novos, Hk, hd, blk, Gq=1, pag=16, camadas=2, sobra=0, e0=-6, solta=(), zera=0.1):
        s = lambda t: R.substream(semente, t)
        self.comp, self.novos, self.Hk, self.hd, self.blk, self.Gq, self.pag, self.camadas = comp, novos, Hk, hd, blk, Gq, pag, camadas
        B, H = len(comp), Hk * Gq
        self.B, self.H, self.gs = B, H, min(hd, blk)
        G = hd // self.gs
        usa = [[(b, p) for p in range(-(-c // pag)) if (b, p) not in solta] for b, c in enumerate(comp)]
        n = sum(map(len, usa)) + 2
        ordem = np.argsort(R.uniform01(s("ordem"), (n,))).tolist()
        forma = (n, camadas, 2, Hk, pag)
        self.m = R.uniform_int(s("lixo"), (*forma, hd), -128, 127).astype(np.int8)
        self.E = R.uniform_int(s("lixoE"), (*forma, G), -128, 127).astype(np.int8)
        self.P = max([-(-c // pag) for c in comp] + [1])
        self.tabela = np.full((B, self.P), -1, np.int32)
        self.ini = np.concatenate([[0], np.cumsum(novos)]).astype(np.int32)
        self.M = int(self.ini[-1]) + sobra
        C = (H + 2 * Hk) * hd
        self.qm, self.qE = R.bloco(s("qkv"), self.M, C, blk, espalha=3, zera=zera, e0=e0)
        for b, paginas in enumerate(usa):
            if not comp[b]:
                continue
            tm, tE = R.bloco(s(f"kv{b}"), comp[b], 2 * Hk * hd, self.gs, espalha=3, zera=zera, e0=e0)
            tm, tE = tm.reshape(comp[b], 2, Hk, hd), tE.reshape(comp[b], 2, Hk, G)
            for _, p in paginas:
                x = self.tabela[b, p] = ordem.pop()
                k = min(pag, comp[b] - p * pag)
                self.m[x, camadas - 1, :, :, :k] = tm[p * pag:p * pag + k].transpose(1, 2, 0, 3)
                self.E[x, camadas - 1, :, :, :k] = tE[p * pag:p * pag + k].transpose(1, 2, 0, 3)

    def incl(self):
        return np.array([2.0 ** -(8 * h // self.H) for h in range(self.H)], np.float32)

    def lote(self, dev, O, com_ini=True):
        return O.Lote(dev(self.tabela), dev(np.array(self.comp, np.int32)), dev(self.ini) if com_ini else None, max(self.novos + [0]), max(self.comp + [0]))

    def escrito(self):
        """The cache after the new rows' keys and values are written."""
        m, E, (H, Hk, hd) = self.m.copy(), self.E.copy(), (self.H, self.Hk, self.hd)
        qm = self.qm.reshape(self.M, H + 2 * Hk, hd)
        col = (np.arange((H + 2 * Hk) * hd // self.gs) * self.gs) // self.blk
        qE = self.qE[:, col].reshape(self.M, H + 2 * Hk, hd // self.gs)
        for b, (c, n) in enumerate(zip(self.comp, self.novos)):
            for t in range(n):
                j, r = c - n + t, self.ini[b] + t
                x = self.tabela[b, j // self.pag]
                m[x, self.camadas - 1, :, :, j % self.pag] = qm[r, H:].reshape(2, Hk, hd)
                E[x, self.camadas - 1, :, :, j % self.pag] = qE[r, H:].reshape(2, Hk, -1)
        return m, E

    def atencao(self, incl=None, janela=0, sumid=0):
        """(output [M, H hd] in float64, what fp32 statistics may be off). The error of one weight exp(u - max) is that of
        its score, 8 roundings of parts no larger than |q| . |k| / sqrt(hd) + incl (i - j) (products are exact), and 8
        more of its own; the sums have at most n + 32 terms, each addition half a unit of a partial sum of |p v|. v and the
        result enter through p (v - o). fp32 ends at 2^-126: a weight below it, next to the largest one's 1, and a product
        or result below it may become 0."""
        H, hd, Gq = self.H, self.hd, self.Gq
        y, tol = np.zeros((self.M, H, hd)), np.zeros((self.M, H, hd))
        q = vale(self.qm, self.qE, self.blk)[:, :H * hd].reshape(self.M, H, hd)
        for b, (c, n) in enumerate(zip(self.comp, self.novos)):
            if n == 0:
                continue
            i, j = np.arange(c - n, c)[:, None], np.arange(c)[None]
            ve = j <= i
            if janela:
                ve &= (j > i - janela) | (j < sumid)
            pg, vaga = self.tabela[b, np.arange(c) // self.pag], np.arange(c) % self.pag
            uso = ve.any(0)
            assert (pg[uso] >= 0).all()
            kv = np.zeros((c, 2, self.Hk, hd))
            kv[uso] = vale(self.m[pg, self.camadas - 1, :, :, vaga], self.E[pg, self.camadas - 1, :, :, vaga], self.gs)[uso]
            r = slice(self.ini[b], self.ini[b] + n)
            for h in range(H):
                k, v = kv[:, 0, h // Gq], kv[:, 1, h // Gq]
                bias = (incl[h] if incl is not None else 0.0) * (i - j)
                u = q[r, h] @ k.T / np.sqrt(hd) - bias
                tam = np.abs(q[r, h]) @ np.abs(k).T / np.sqrt(hd) + np.abs(bias)
                u = np.where(ve, u, -np.inf)
                p = np.exp(u - u.max(1, keepdims=True))
                p /= p.sum(1, keepdims=True)
                o = p @ v
                y[r, h] = o
                rel = p * np.where(ve, 8 * tam + 8, 0.0)
                conta = ve.sum(1, keepdims=True) + 32
                tol[r, h] = 2.0 ** -24 * (rel @ np.abs(v) + rel.sum(1, keepdims=True) * np.abs(o) + conta * (p @ np.abs(v) + np.abs(o))) + 2.0 ** -126 * (ve @ np.abs(v) + ve.sum(1, keepdims=True) + 1)
        return y.reshape(self.M, -1), tol.reshape(self.M, -1)
