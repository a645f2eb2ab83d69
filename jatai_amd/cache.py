"""A paged cache of keys and values for generation (no reference counterpart: the reference only trains).

The pages live in HBM as one block tensor (m int8 [pages, layers, 2, heads, slots, width], E int8 [.., exponents per
head]; `CacheKV.C`, what `OpsHip.cache_grava` and `OpsHip.atencao_cache` take). A page holds the keys and values of
`pagina` consecutive tokens of a sequence in every layer, so one table serves them all. Which page holds what is kept on
the host, where every length is known before a step runs; the kernels read the tables from `tabela` and `comp`, device
tensors at fixed addresses, which a captured graph follows. Pages are counted by their holders: a fork shares the pages
of its origin, and whoever writes first into a shared page gets a copy of it.
"""
import heapq

import torch

from . import ops as O


class CacheKV:
    def __init__(self, ops, camadas, cabecas, hd, paginas, seqs, max_tokens, pagina=64, dev="cuda"):
        """paginas pages of `pagina` slots for `camadas` layers of `cabecas` heads of width hd; up to `seqs` sequences of
        max_tokens tokens each."""
        self.ops, self.reg, self.pagina, self.max_tokens = ops, ops.reg, pagina, max_tokens
        self.reg.exige(min(camadas, cabecas, paginas, seqs, max_tokens) > 0 and hd in (4, 16, 32, 64, 128) and pagina in (16, 32, 64, 128, 256, 512, 1024),
                       f"CacheKV: {camadas} camadas, {cabecas} cabecas de {hd} (4, 16, 32, 64 ou 128), {paginas} paginas de {pagina} (potencia de 2 de 16 a 1024), "
                       f"{seqs} sequencias de {max_tokens} tokens")
        P = -(-max_tokens // pagina)
        self.C = (torch.zeros(paginas, camadas, 2, cabecas, pagina, hd, dtype=torch.int8, device=dev),
                  torch.zeros(paginas, camadas, 2, cabecas, pagina, hd // min(hd, O.BLK), dtype=torch.int8, device=dev))
        self.tabela = torch.full((seqs, P), -1, dtype=torch.int32, device=dev)
        self.comp = torch.zeros(seqs, dtype=torch.int32, device=dev)
        self.n = [0] * seqs                       # tokens of each sequence
        self.paginas = [[] for _ in range(seqs)]  # its pages in order; -1 where esquece let one go
        self.usos = [0] * paginas
        self._livres = list(range(paginas))       # a heap: the lowest free page is handed out first
        self._mudou = True

    @property
    def livres(self):
        return len(self._livres)

    def _seq(self, op, *seqs):
        if not all(isinstance(s, int) and 0 <= s < len(self.n) for s in seqs):
            self.reg.falha(f"{op}: sequencias {seqs}, de 0 a {len(self.n) - 1}")

    def _larga(self, p):
        if p >= 0:
            self.usos[p] -= 1
            if self.usos[p] == 0:
                heapq.heappush(self._livres, p)

    def _pega(self):
        p = heapq.heappop(self._livres)
        self.usos[p] = 1
        return p

    def reserva(self, novos):
        """Room for the new tokens of a step, novos = {sequence: tokens}: their lengths grow, pages are taken, and a
        page that would be written while others hold it is copied first. Where pages or room are short nothing changes."""
        self._seq("reserva", *novos)
        falta, copias = 0, []
        for s, k in novos.items():
            if k < 0 or self.n[s] + k > self.max_tokens:
                self.reg.falha(f"reserva: sequencia {s} com {self.n[s]} + {k} tokens, ate {self.max_tokens}")
            falta += -(-(self.n[s] + k) // self.pagina) - len(self.paginas[s])
            if k and self.n[s] % self.pagina:
                p = self.paginas[s][-1]
                if p < 0:
                    self.reg.falha(f"reserva: a ultima pagina da sequencia {s} foi esquecida")
                copias.append((s, p))
        # the holders of a shared page that write it now: all but the last to go take a copy, the last only if it stays shared
        fica = {}
        for s, p in copias:
            fica[p] = fica.get(p, self.usos[p]) - 1
        tira = {p: self.usos[p] - 1 if r == 0 else self.usos[p] - r for p, r in fica.items()}   # copies each page needs
        if falta + sum(tira.values()) > self.livres:
            self.reg.falha(f"reserva: faltam paginas ({falta + sum(tira.values())} pedidas, {self.livres} livres)")
        pares = []
        for s, p in copias:
            if tira[p]:
                tira[p] -= 1
                self.paginas[s][-1] = self._pega()
                pares.append((p, self.paginas[s][-1]))
                self._larga(p)
                self._mudou = True
        for s, k in novos.items():
            self.n[s] += k
            while len(self.paginas[s]) * self.pagina < self.n[s]:
                self.paginas[s].append(self._pega())
                self._mudou = True
        if pares:
            self.ops.cache_copia(self.C, pares)

    def bifurca(self, de, para):
        """Sequence `para` (empty) becomes a fork of `de`: it shares its pages, copied only when one of them writes."""
        self._seq("bifurca", de, para)
        if de == para or self.n[para] or self.paginas[para]:
            self.reg.falha(f"bifurca: {de} -> {para} ({self.n[para]} tokens; o destino deve estar vazio)")
        self.n[para], self.paginas[para] = self.n[de], list(self.paginas[de])
        for p in self.paginas[de]:
            if p >= 0:
                self.usos[p] += 1
        self._mudou = True

    def libera(self, seq):
        """The sequence is empty again; pages that nobody else holds are free."""
        self._seq("libera", seq)
        for p in self.paginas[seq]:
            self._larga(p)
        self.n[seq], self.paginas[seq], self._mudou = 0, [], True

    def esquece(self, seq, janela, sumidouros=0):
        """Lets go of the pages that no later token of the sequence sees with this window: those that hold neither one of
        the last janela - 1 tokens nor one of the first `sumidouros`."""
        self._seq("esquece", seq)
        if janela <= 0 or sumidouros < 0:
            self.reg.falha(f"esquece: janela={janela}, sumidouros={sumidouros}")
        fim = self.n[seq] + 1 - janela             # the next token sees from here on
        for i, p in enumerate(self.paginas[seq]):
            if (i + 1) * self.pagina > fim:
                break
            if p >= 0 and i * self.pagina >= sumidouros:
                self._larga(p)
                self.paginas[seq][i] = -1
                self._mudou = True

    def compacta(self):
        """Moves the pages in use to the lowest numbers; returns the number of pages moved. Every holder of a page follows."""
        usadas = sum(u > 0 for u in self.usos)
        de = [p for p in range(usadas, len(self.usos)) if self.usos[p]]
        para = [p for p in range(usadas) if not self.usos[p]]
        if not de:
            return 0
        self.ops.cache_copia(self.C, list(zip(de, para)))
        mapa = dict(zip(de, para))
        self.paginas = [[mapa.get(p, p) for p in ps] for ps in self.paginas]
        for a, b in mapa.items():
            self.usos[b], self.usos[a] = self.usos[a], 0
        self._livres = list(range(usadas, len(self.usos)))
        self._mudou = True
        return len(de)

    def envia(self, comprimentos=True):
        """Tables (only if they changed) and lengths to the device tensors."""
        if self._mudou:
            P = self.tabela.shape[1]
            self.tabela.copy_(torch.tensor([ps + [-1] * (P - len(ps)) for ps in self.paginas], dtype=torch.int32))
            self._mudou = False
        if comprimentos:
            self.comp.copy_(torch.tensor(self.n, dtype=torch.int32))

    def lote(self, novos, ini=None, teto=None):
        """The Lote of all sequences: at most `novos` new tokens each, whose rows start at ini (None: row s is sequence
        s's), none longer than teto (None: max_tokens)."""
        return O.Lote(self.tabela, self.comp, ini, novos, self.max_tokens if teto is None else teto)
