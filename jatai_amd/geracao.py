"""Continuing text with a trained model (no reference counterpart: the reference only trains): the forward pass of
`Modelo.passo` for new tokens only, their attention over a paged cache of everything before them.

Prompts of any lengths run as the rows of one batch; a step of one token per sequence is captured as a hipGraph and
replayed. Products, norms and residual adds are the training step's own (or gemv4 on weights packed to 4 bits); the
attention is `OpsHip.atencao_cache`, softmax in float32 over exact products, with the training's position bias.
Where the training attention aligns a whole window to one exponent and rounds its weights to 8 bits, this one rounds
only its output, so that a token's result does not depend on what comes later and lengths are not bound to 512.
"""
import weakref

import torch

from . import ops as O
from .cache import CacheKV

# generators with steps whose device events have not been read: the device holds one record for all, which is cleared only when
# nobody has any left to read
_pendentes = weakref.WeakSet()


class Gerador:
    def __init__(self, modelo, seqs, max_tokens, pagina=64, paginas=None, bits=8, janela=0, sumidouros=0):
        """Up to `seqs` sequences of max_tokens tokens. bits: 8 runs the model's own weights, 4 packs them once (para4).
        janela > 0: attention to the last `janela` tokens and the first `sumidouros`; pages in between are let go.
        paginas: pages of the cache (None: enough for every sequence's max_tokens)."""
        self.m, self.ops, self.reg = modelo, modelo.ops, modelo.reg
        self.reg.exige(bits in (4, 8) and seqs > 0 and max_tokens > 0, f"Gerador: bits={bits} (4 ou 8), seqs={seqs}, max_tokens={max_tokens}")
        self.bits, self.janela, self.sumidouros, self.seqs = bits, janela, sumidouros, seqs
        hd = modelo.D // modelo.H
        P = -(-max_tokens // pagina)
        self.cache = CacheKV(self.ops, modelo.L, modelo.H, hd, seqs * P if paginas is None else paginas, seqs, max_tokens, pagina, modelo.dev)
        self.incl = self.ops.inclinacoes(modelo.H, hd, modelo.dev)
        self.w = {n: self.ops.para4(t) for n, t in modelo.p.items() if n != "emb"} if bits == 4 else modelo.p
        # a step's rows: one per sequence, padded to the 32 that the 8-bit products take; rows of idle ones come to nothing
        self.linhas = seqs if bits == 4 else -(-seqs // 32) * 32
        z = lambda n: torch.zeros(n, dtype=torch.int32, device=modelo.dev)
        self.tok, self.vivas, self.comp, self._grafo, self.lancamentos = z(self.linhas), z(seqs), z(seqs), None, []
        self._indices = torch.arange(modelo.V, dtype=torch.int32, device=modelo.dev)
        self._estado = None                        # (live sequences, their lengths) as the device tensors hold them

    # ------------------------------------------------------------------ the forward pass of new tokens
    def _produto(self, X, n):
        return self.ops.gemv4(X, self.w[n]) if self.bits == 4 else self.ops.gemm(X, self.w[n])

    def _camadas(self, tok, lote, ultimas=None):
        """Raw logits of the rows `ultimas` (all of them when None) of the tokens tok [M]."""
        ops, m, quatro, r16 = self.ops, self.m, self.bits == 4, self.m.r16
        with self.reg.trecho("embedding"):
            x = ops.embed(m.p["emb"], tok)
            x16 = ops.para16(x) if r16 else None
        for l in range(m.L):
            with self.reg.trecho(f"camada {l}"):
                with self.reg.trecho("atencao"):
                    qkv = self._produto(ops.rms(x)[0], f"Wqkv{l}")
                    ops.cache_grava(qkv, self.cache.C, l, lote)
                    om = ops.atencao_cache(qkv, self.cache.C, l, lote, self.incl, self.janela, self.sumidouros)
                    if r16:
                        x16 = ops.soma16(x16, self._produto(om, f"Wo{l}"))
                        x = ops.para8(x16)
                    else:
                        x = ops.gemv4_soma(om, self.w[f"Wo{l}"], x) if quatro else ops.gemm_soma(om, self.w[f"Wo{l}"], x)
                with self.reg.trecho("mlp"):
                    n2 = ops.rms(x)[0]
                    a = ops.gemv4_relu2(n2, self.w[f"Wup{l}"]) if quatro else ops.gemm_relu2(n2, self.w[f"Wup{l}"])[1]
                    if r16:
                        x16 = ops.soma16(x16, self._produto(a, f"Wd{l}"))
                        x = ops.para8(x16)
                    else:
                        x = ops.gemv4_soma(a, self.w[f"Wd{l}"], x) if quatro else ops.gemm_soma(a, self.w[f"Wd{l}"], x)
        with self.reg.trecho("saida"):
            nf = ops.rms(x)[0]
            if ultimas is not None:
                nf = nf[0][ultimas], nf[1][ultimas]
            return ops.valores(ops.gemv4(nf, self.w["out"], cru=True) if quatro else ops.gemm(nf, self.w["out"], cru=True))

    def _mais_provavel(self, y):
        """The index of each row's largest logit, the lowest of equals."""
        return torch.where(y == y.amax(1, keepdim=True), self._indices, self.m.V - 1).amin(1)

    def _esquece(self):
        if self.janela > 0:
            for s in range(self.seqs):
                self.cache.esquece(s, self.janela, self.sumidouros)

    def le(self, textos):
        """New tokens for some sequences, textos = {sequence: tokens (at least one)}: prompts, or continuations of what the
        cache holds. Returns the logits after each one's last token, float32 [len(textos), V] in textos' order. An error leaves
        the sequences it was called for with nothing of use: free them."""
        reg, V = self.reg, self.m.V
        reg.exige(len(textos) > 0 and all(len(t) > 0 for t in textos.values()), "le: cada sequencia com pelo menos um token")
        reg.exige(all(0 <= x < V for t in textos.values() for x in t), f"le: tokens de 0 a {V - 1}")
        for g in list(_pendentes):
            g.confere()
        reg.novo_passo(reg.passo)
        self.cache.reserva({s: len(t) for s, t in textos.items()})
        self.cache.envia()
        plano, ini, ultima = [], [0], {}
        for s in range(self.seqs):                 # rows in the order of the sequences
            plano += list(textos.get(s, ()))
            ini.append(len(plano))
            ultima[s] = len(plano) - 1
        M = len(plano) if self.bits == 4 else -(-len(plano) // 32) * 32
        dev = self.m.dev
        tok = torch.tensor(plano + [0] * (M - len(plano)), dtype=torch.int32).to(dev)
        quais = [ultima[s] for s in textos]
        quais += [quais[0]] * (0 if self.bits == 4 else -len(quais) % 32)
        lote = self.cache.lote(max(map(len, textos.values())), torch.tensor(ini, dtype=torch.int32).to(dev), max(self.cache.n))
        with reg.trecho("le"):
            y = self._camadas(tok, lote, torch.tensor(quais).to(dev))[:len(textos)]
        reg.fim_passo()
        self._esquece()
        return y

    def confere(self):
        """Reads the device events of the steps so far (waits for them); one that was raised becomes an ErroJatai. Comes before
        training steps or other work that clears the device's record; of several generators with steps to read each one raises."""
        if self in _pendentes:
            _pendentes.discard(self)
            self.reg.lancamentos = self.lancamentos
            self.reg.fim_passo()

    # ------------------------------------------------------------------ one token per sequence, captured
    def _grava(self):
        """The step as a hipGraph: the live sequences grow by one, their tokens run through the layers, and each one's most
        likely next token (the lowest of equals) is chosen. Lengths, tables and tokens are read when it runs."""
        torch.cuda.synchronize()
        anterior, self.reg.lancamentos = self.reg.lancamentos, []
        grafo, lib = torch.cuda.CUDAGraph(), self.ops.lib
        vigiar, self.reg.vigiar = self.reg.vigiar, False
        try:
            with torch.cuda.graph(grafo):
                lib.jt_stream(torch.cuda.current_stream().cuda_stream)
                self.comp.add_(self.vivas)
                with self.reg.trecho("passo"):
                    lote = O.Lote(self.cache.tabela, self.comp, None, 1, self.cache.max_tokens)
                    self.logits = self._camadas(self.tok, lote)[:self.seqs]
                self.escolha = self._mais_provavel(self.logits)
        finally:
            lib.jt_stream(None)
            self.reg.vigiar = vigiar
            self.lancamentos, self.reg.lancamentos = list(self.reg.lancamentos), anterior
        self._grafo = grafo

    def passo(self, vivas, tok):
        """One token for each of the sequences `vivas`: tok, an int32 tensor [seqs] on the device (the others' are not read).
        Returns (logits float32 [seqs, V], the most likely next tokens int32 [seqs]), the graph's own tensors, which
        the next step overwrites; rows of other sequences hold nothing of use. Does not wait: confere() reads events."""
        self.reg.exige(tok.dtype == torch.int32 and tuple(tok.shape) == (self.seqs,) and tok.is_cuda, f"passo: tok int32 {(self.seqs,)} na GPU")
        vivas = sorted(vivas)
        self.reg.exige(len(set(vivas)) == len(vivas), f"passo: sequencia repetida em {vivas}")
        if self._grafo is None:
            self._grava()
        if not _pendentes:
            self.reg.novo_passo(self.reg.passo)
        self.cache.reserva({s: 1 for s in vivas})
        estado = (vivas, [self.cache.n[s] - 1 for s in vivas])
        if self._estado != estado:
            comp, mascara = [0] * self.seqs, [0] * self.seqs
            for s, n in zip(*estado):
                comp[s], mascara[s] = n, 1
            self.comp.copy_(torch.tensor(comp, dtype=torch.int32))
            self.vivas.copy_(torch.tensor(mascara, dtype=torch.int32))
        self.cache.envia(comprimentos=False)
        self.tok[:self.seqs].copy_(tok)
        self._grafo.replay()
        self._estado = (vivas, [n + 1 for n in estado[1]])
        _pendentes.add(self)
        self.reg.lancamentos = list(self.lancamentos)
        self._esquece()
        return self.logits, self.escolha

    def gera(self, textos, n, escolhe=None):
        """Continues each text (a list of tokens) by n tokens; returns the lists of new ones. escolhe(logits float32 [k, V])
        gives the k next tokens (None: the most likely). Uses sequences that are empty, and frees them."""
        livres = [s for s in range(self.seqs) if self.cache.n[s] == 0]
        self.reg.exige(len(textos) <= len(livres) and n >= 0, f"gera: {len(textos)} textos, {len(livres)} sequencias livres, n={n}")
        if not textos or n == 0:
            return [[] for _ in textos]
        quais = livres[:len(textos)]
        onde = torch.tensor(quais).to(self.m.dev)
        escolhe = escolhe or self._mais_provavel
        tok = torch.zeros(self.seqs, dtype=torch.int32, device=self.m.dev)
        saida = []
        try:
            y = self.le(dict(zip(quais, textos)))
            while True:
                novos = escolhe(y).to(torch.int32)
                saida.append(novos)
                if len(saida) == n:
                    break
                tok[onde] = novos
                y = self.passo(quais, tok)[0][onde]
            self.confere()
        finally:
            for s in quais:
                self.cache.libera(s)
        return torch.stack(saida, 1).tolist()
