"""Performance cases of the operators that let a trained model answer: attention of new tokens over a paged key-value
cache, the cache's own page operators, and products of a few rows with 4-bit weights. Each case is one call of a user's
program; `run` makes it in plain torch (`own` false) or through `jatai_amd` (`own` true).

The formats are the framework's: a block tensor is int8 mantissas [R, C] and int8 exponents [R, C / blk], value m 2^E; a
raw tensor is int32 mantissas and int16 exponents, one each per value. The cache is a pair of tensors [pages, layers, 2
(keys, values), heads, slots, width] and [.., groups] (a group: the values of a head that share an exponent).
"""
import math
import os
import tempfile

import torch

own = False

DEV = "cuda"
E_ZERO = -127


def listed():
    return [
        # one sequence's next token, a short conversation: the smallest call, where only latency counts
        dict(name="token_1_seq", tipo="atencao", B=1, H=8, Hk=8, hd=64, blk=32, pag=64, cmin=200, cmax=200, nmin=1, nmax=1, janela=0, sumid=0, saida="bf16", camadas=12),
        # the next tokens of a batch of models of the reference's own shape (64 heads of 4, blocks of 128), ragged contexts
        dict(name="token_16_seq_cab4", tipo="atencao", B=16, H=64, Hk=64, hd=4, blk=128, pag=64, cmin=37, cmax=2050, nmin=1, nmax=1, janela=0, sumid=0, saida="bloco", camadas=12),
        # a few very long contexts: the work is split over the cache's length
        dict(name="token_longo", tipo="atencao", B=4, H=8, Hk=8, hd=64, blk=32, pag=64, cmin=90001, cmax=131071, nmin=1, nmax=1, janela=0, sumid=0, saida="bf16", camadas=1),
        # a full batch whose query heads share key-value heads
        dict(name="token_64_seq_grupos", tipo="atencao", B=64, H=32, Hk=8, hd=128, blk=32, pag=64, cmin=500, cmax=4096, nmin=1, nmax=1, janela=0, sumid=0, saida="bf16", camadas=1),
        # a batch far past its window: 1024 tokens and the first 4 stay visible, pages in between are freed
        dict(name="token_janela", tipo="atencao", B=64, H=8, Hk=8, hd=64, blk=32, pag=64, cmin=300, cmax=16384, nmin=1, nmax=1, janela=1024, sumid=4, saida="f32", camadas=1),
        # prompts of different lengths in one call: every token is new
        dict(name="prompts", tipo="atencao", B=8, H=8, Hk=8, hd=64, blk=32, pag=64, cmin=1, cmax=4000, nmin=1, nmax=4000, janela=0, sumid=0, saida="bloco", camadas=1),
        # a step's keys and values written into the pages, one token per sequence
        dict(name="grava_token", tipo="grava", B=32, H=8, Hk=8, hd=64, blk=32, pag=64, cmin=1, cmax=250, nmin=1, nmax=1, camadas=1),
        # the keys and values of prompts
        dict(name="grava_prompts", tipo="grava", B=16, H=8, Hk=8, hd=64, blk=32, pag=64, cmin=300, cmax=2048, nmin=300, nmax=2048, camadas=1),
        # one page of all 12 layers copied when a fork of a sequence first writes
        dict(name="copia_1", tipo="copia", pares=1, paginas=8, Hk=8, hd=64, blk=32, pag=64, camadas=12),
        # a cache compacted: many pages moved
        dict(name="compacta", tipo="copia", pares=300, paginas=640, Hk=8, hd=64, blk=32, pag=64, camadas=12),
        # the Q/K/V product of one token of the 12-layer model, 4-bit weights, raw output
        dict(name="gemv4_1", tipo="gemv4", modo="cru", M=1, N=1536, K=512, blk=32),
        # one product of a large model's step, 16 sequences
        dict(name="gemv4_16", tipo="gemv4", modo="cru", M=16, N=8192, K=8192, blk=32),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    tipo = rng.choice(["atencao", "atencao", "atencao", "grava", "copia", "gemv4", "gemv4"])
    blk = rng.choice([32, 32, 128])
    if tipo == "gemv4":
        modo = rng.choice(["cru", "cru", "soma", "relu2"])
        K = blk * max(1, round(_log(rng, 128, 8192) / blk))
        N = _log(rng, 32, 8192)
        N = N if modo == "cru" else blk * max(1, round(N / blk))
        return dict(tipo=tipo, modo=modo, M=_log(rng, 1, 64), N=N, K=K, blk=blk)
    hd = rng.choice([64, 64, 128, 32, 16, 4])
    Hk = rng.choice([32, 64]) if hd == 4 else rng.choice([h for h in (2, 4, 6, 8, 12, 16) if h * hd % 128 == 0 and h * hd <= 1024])
    pag = rng.choice([16, 32, 64, 64, 128])
    if tipo == "copia":
        camadas = rng.choice([1, 2, 12])
        pares = min(_log(rng, 1, 300), max(1, 240_000_000 // (2 * Hk * hd * pag * camadas)))
        return dict(tipo=tipo, pares=pares, paginas=2 * pares + rng.randint(1, 40), Hk=Hk, hd=hd, blk=blk, pag=pag, camadas=camadas)
    H = Hk * (1 if hd == 4 else rng.choice([1, 1, 1, 2, 4]))
    B = _log(rng, 1, 64)
    if tipo == "grava":
        passo = rng.random() < 0.5
        cmax = _log(rng, 1, 32768 // B)
        cmin = rng.randint(1, cmax)
        return dict(tipo=tipo, B=B, H=H, Hk=Hk, hd=hd, blk=blk, pag=pag, cmin=cmin, cmax=cmax, nmin=1 if passo else rng.randint(0, cmin),
                    nmax=1 if passo else cmax, camadas=rng.choice([1, 2]))
    forma = rng.choice(["token", "token", "token", "prompts", "trecho"])
    cmax = _log(rng, 1, 131072 // B if forma == "token" else (4000 if H * hd <= 1024 else 2000) // B)
    cmin = rng.randint(1, cmax)
    nmin, nmax = dict(token=(1, 1), prompts=(cmin, cmax), trecho=(0 if B > 1 else 1, min(cmin, rng.randint(2, 40))))[forma]
    janela = rng.choice([0, 0, _log(rng, 1, 4096)])
    return dict(tipo=tipo, B=B, H=H, Hk=Hk, hd=hd, blk=blk, pag=pag, cmin=cmin, cmax=cmax, nmin=nmin, nmax=nmax, janela=janela,
                sumid=rng.choice([0, 1, 4, 70]) if janela else 0, saida=rng.choice(["bf16", "bf16", "f32", "bloco"]), camadas=rng.choice([1, 2]))


# ------------------------------------------------------------------------------------------------ inputs
def _comprimentos(c):
    """Tokens in the cache of each sequence and how many of them are new: spread evenly over the case's ranges."""
    B = c["B"]
    passo = lambda lo, hi: [lo + (hi - lo) * b // max(B - 1, 1) for b in range(B)]
    comp = passo(c["cmin"], c["cmax"])
    return comp, [min(n, x) for n, x in zip(passo(c["nmin"], c["nmax"]), comp)]


def _bloco(x, blk):
    """x [R, C] in the block format: one exponent per blk columns, E = (binary exponent of the largest value) - 7, one
    higher where a rounded mantissa passes 127, half to even; a zero block, or one below 2^-126, has E = -127."""
    R, C = x.shape
    v = x.view(R, C // blk, blk)
    maior = v.abs().amax(2, keepdim=True)
    E = torch.frexp(maior)[1] - 7
    escala = lambda E: torch.ldexp(torch.ones_like(maior), -E)
    E = E + (torch.round(maior * escala(E)) > 127)
    zero = (maior == 0) | (E < -126)
    q = torch.where(zero, torch.zeros_like(v), torch.round(v * escala(E)))
    return q.view(R, C).to(torch.int8), torch.where(zero, torch.full_like(E, E_ZERO), E).view(R, C // blk).to(torch.int8)


def _normal(g, R, C, blk, sigma=1.0):
    """N(0, sigma^2) values, rows scaled by a log-normal factor as the activations of different tokens are."""
    x = torch.randn(R, C, generator=g, device=DEV) * sigma
    return _bloco(x * torch.exp(0.5 * torch.randn(R, 1, generator=g, device=DEV)), blk)


def _grupos(c):
    """Values of a head that share an exponent, and such groups per head."""
    gs = min(c["hd"], c["blk"])
    return gs, c["hd"] // gs


def _paginas(g, c, n, valido=None):
    """n pages of keys and values as a model writes them; where `valido` [n, slots] is false, what memory happened to hold."""
    gs, G = _grupos(c)
    forma = (n, c["camadas"], 2, c["Hk"], c["pag"])
    m = torch.empty(*forma, c["hd"], dtype=torch.int8, device=DEV)
    E = torch.empty(*forma, G, dtype=torch.int8, device=DEV)
    m.random_(-127, 128, generator=g)
    E.random_(-9, -4, generator=g)
    if valido is not None:
        livre = ~valido.view(n, 1, 1, 1, c["pag"], 1)
        m = torch.where(livre, torch.full_like(m, -128), m)
        E = torch.where(livre, torch.empty_like(E).random_(-128, 128, generator=g), E)
    return m, E


def _inclinacoes(c):
    """The framework's position bias per query head, in nats per token of distance."""
    H, hd = c["H"], c["hd"]
    incl = [8 - h // 8 if hd == 4 else 8 - 8 * h // H for h in range(H)]
    return torch.tensor([2.0 ** (i - 8) if i >= 0 else 0.0 for i in incl], dtype=torch.float32, device=DEV)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case=c)
    if c["tipo"] == "gemv4":
        return _prepara_gemv4(c, g, s)
    if c["tipo"] == "copia":
        s["cache"] = _paginas(g, c, c["paginas"])
        ordem = torch.randperm(c["paginas"], generator=g, device=DEV).tolist()
        s["pares"] = list(zip(ordem[:c["pares"]], ordem[c["pares"]:2 * c["pares"]]))
        return s
    # ragged sequences over a shuffled page table; table entries behind a sequence, and pages that its window has left
    # behind, hold -1
    comp, novos = _comprimentos(c)
    ordem = torch.randperm(c["B"], generator=g, device=DEV).tolist()
    comp, novos = [comp[i] for i in ordem], [novos[i] for i in ordem]
    pag, janela, sumid = c["pag"], c.get("janela", 0), c.get("sumid", 0)
    usa = []
    for L, n in zip(comp, novos):
        visivel = lambda p: not janela or p * pag < sumid or (p + 1) * pag > L - max(n, 1) + 1 - janela
        usa.append([p if visivel(p) else -1 for p in range(-(-L // pag))])
    largura, total = max(len(u) for u in usa), sum(p >= 0 for u in usa for p in u)
    paginas = torch.randperm(total + 3, generator=g, device=DEV)[:total].to(torch.int32).tolist()
    tabela, valido = [], torch.zeros(total + 3, pag, dtype=torch.bool)
    for u, L, n in zip(usa, comp, novos):
        linha = [-1 if p < 0 else paginas.pop() for p in u]
        for p, x in zip(u, linha):
            if x >= 0:
                valido[x, :min(pag, L - p * pag)] = True
        tabela.append(linha + [-1] * (largura - len(linha)))
    ini = [0]
    for n in novos:
        ini.append(ini[-1] + n)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    linhas = max(1, ini[-1]) if c["nmax"] == 1 else -(-max(ini[-1], 1) // 32) * 32       # prompts: padded to the products' 32 rows
    D, Dk = c["H"] * c["hd"], c["Hk"] * c["hd"]
    qkv = torch.cat([torch.randn(linhas, D, generator=g, device=DEV) * 1.5, torch.randn(linhas, 2 * Dk, generator=g, device=DEV)], 1)
    qkv = qkv * torch.exp(0.3 * torch.randn(linhas, 1, generator=g, device=DEV))
    s.update(qkv=_bloco(qkv, c["blk"]), cache=_paginas(g, c, total + 3, valido.to(DEV)), tabela=i32(tabela), comp=i32(comp), ini=i32(ini),
             novos=max(novos), teto=max(comp), incl=_inclinacoes(c))
    return s


def _prepara_gemv4(c, g, s):
    """4-bit weights with one scale per row and group of blk columns, as a program packs them once: per row the exponent
    R of its largest scale, scales relative to it (an 8-bit mantissa each, exact in bfloat16), weights in [-7, 7]."""
    M, N, K, blk = c["M"], c["N"], c["K"], c["blk"]
    w = torch.randn(N, K, generator=g, device=DEV) * torch.exp(0.4 * torch.randn(N, 1, generator=g, device=DEV)) * K ** -0.5
    w = w.view(N, K // blk, blk)
    f, e = torch.frexp(w.abs().amax(2) / 7)
    s8 = torch.round(f * 256)                                          # 128 .. 256
    e = torch.where(s8 > 255, e + 1, e) - 8
    s8 = torch.where(s8 > 255, s8 / 2, s8)
    q = torch.round(w / (s8 * torch.exp2(e.float())).unsqueeze(2)).clamp(-7, 7).to(torch.int32).view(N, K)
    R = e.amax(1)
    esc = (s8 * torch.exp2((e - R.unsqueeze(1)).float())).to(torch.bfloat16)
    s["W"] = (*_empacota(q, esc, blk), R.to(torch.int16))
    s["x"] = _normal(g, M, K, blk)
    if c["modo"] == "soma":
        s["res"] = _normal(g, M, N, blk)
    return s


def _empacota(q, esc, blk):
    """The packed layout: tiles of 16 rows x 128 columns, 1024 bytes each. Byte 4 a + i of lane l (a: the group of 32
    columns, i: 0 .. 3) holds row l % 16's columns 32 a + 8 (l // 16) + i (low four bits) and + 4 (high), two's
    complement; the scales [N / 16, K / 128, 16, groups]. Missing rows and columns are zeros."""
    N, K = q.shape
    Nt, Kt, G = -(-N // 16), -(-K // 128), 128 // blk
    cheio = torch.zeros(Nt * 16, Kt * 128, dtype=torch.int32, device=q.device)
    cheio[:N, :K] = q
    t = cheio.view(Nt, 16, Kt, 4, 4, 2, 4).permute(0, 2, 4, 1, 3, 6, 5)  # tile, tile, l // 16, l % 16, a, i, half
    m = ((t[..., 0] & 15) | ((t[..., 1] & 15) << 4)).to(torch.uint8).reshape(Nt, Kt, 64, 16)
    e = torch.zeros(Nt * 16, Kt * G, dtype=torch.bfloat16, device=q.device)
    e[:N, :esc.shape[1]] = esc
    return m.contiguous(), e.view(Nt, 16, Kt, G).permute(0, 2, 1, 3).contiguous()


# ------------------------------------------------------------------------------------------------ one pass
_OPS = {}


def _ops(blk):
    """The program's operator object: one per process, at the program's block size. A step's launch list is dropped before
    the next step's (the device's error record is cleared and read once per step of all layers, not per operator)."""
    from jatai_amd import ops as O
    if not _OPS:
        from jatai_amd.registro import Registro
        _OPS["reg"] = Registro(os.path.join(tempfile.gettempdir(), "jatai_perf"), "operadores", eco=False)
        _OPS["ops"] = O.OpsHip(_OPS["reg"])
    O.BLK = blk
    _OPS["reg"].lancamentos = []
    return _OPS["ops"], O


def run(state):
    c = state["case"]
    if own:
        return globals()["_chama_" + c["tipo"]](c, state, *_ops(c["blk"]))
    return globals()["_" + c["tipo"]](c, state)


def _lote(s, O):
    return O.Lote(s["tabela"], s["comp"], s["ini"], s["novos"], s["teto"])


def _chama_atencao(c, s, ops, O):
    saida = dict(bf16=torch.bfloat16, f32=torch.float32, bloco=None)[c["saida"]]
    y = ops.atencao_cache(s["qkv"], s["cache"], c["camadas"] - 1, _lote(s, O), incl=s["incl"], janela=c["janela"], sumidouros=c["sumid"], saida=saida)
    return ops.valores(y, torch.bfloat16) if saida is None else y


def _chama_grava(c, s, ops, O):
    return ops.cache_grava(s["qkv"], s["cache"], c["camadas"] - 1, _lote(s, O))


def _chama_copia(c, s, ops, O):
    return ops.cache_copia(s["cache"], s["pares"])


def _chama_gemv4(c, s, ops, O):
    if c["modo"] == "cru":
        return ops.gemv4(s["x"], s["W"], cru=True)
    return ops.valores(ops.gemv4_soma(s["x"], s["W"], s["res"]) if c["modo"] == "soma" else ops.gemv4_relu2(s["x"], s["W"]), torch.bfloat16)


# ------------------------------------------------------------------------------------------------ the plain forms
def _vale(m, E, n):
    """The values of mantissas whose last axis is shared out among the exponents' in runs of n."""
    f = torch.exp2(E.float()).unsqueeze(-1)
    return (m.unflatten(-1, (-1, n)).float() * f).flatten(-2)


def _linhas(s):
    """Sequence and position of every row of the batch; rows behind the last sequence have sequence -1."""
    r = torch.arange(s["qkv"][0].shape[0], device=DEV)
    ini = s["ini"].long()
    b = torch.searchsorted(ini, r, right=True) - 1
    fora = r >= ini[-1]
    b = torch.where(fora, 0, b)
    return torch.where(fora, -1, b), s["comp"].long()[b] - (ini[b + 1] - r)


def _atencao(c, s):
    """softmax(q . k / sqrt(hd) - incl (i - j)) v over the visible tokens j <= i of each row's sequence (the last `janela`
    of them and the first `sumid`), in float32; a row without any gives zeros."""
    H, Hk, hd, blk, pag = c["H"], c["Hk"], c["hd"], c["blk"], c["pag"]
    gs, _ = _grupos(c)
    m, E = s["cache"]
    b, pos = _linhas(s)
    M, L, B, camada = b.numel(), s["teto"], c["B"], c["camadas"] - 1
    j = torch.arange(L, device=DEV)
    pg = s["tabela"][:, j // pag].long().clamp(min=0)                                   # [B, L]
    kv = _vale(m[pg, camada, :, :, j % pag], E[pg, camada, :, :, j % pag], gs)           # [B, L, 2, Hk, hd]
    q = _vale(s["qkv"][0], s["qkv"][1], blk)[:, :H * hd].view(M, H, hd)
    # rows of one sequence side by side: [B, n, ..], padded
    n = max(s["novos"], 1)
    linha = s["ini"][:-1].long().unsqueeze(1) + torch.arange(n, device=DEV)
    tem = linha < s["ini"][1:].long().unsqueeze(1)
    linha = torch.where(tem, linha, 0)
    qb = q[linha].view(B, n, Hk, H // Hk, hd).permute(0, 2, 1, 3, 4).reshape(B * Hk, n * (H // Hk), hd)
    kb = kv[:, :, 0].permute(0, 2, 3, 1).reshape(B * Hk, hd, L)
    i = torch.where(tem, pos[linha], -1).view(B, 1, n, 1, 1)
    vis = (j <= i) & ((j > i - c["janela"]) | (j < c["sumid"]) if c["janela"] else (j == j))
    # masked keys may hold anything, infinities among it: replaced before they are used
    usada = vis.view(B, n, L).any(1)
    kb = torch.where(usada.view(B, 1, 1, L), kb.view(B, Hk, hd, L), 0.0).view(B * Hk, hd, L)
    vb = torch.where(usada.view(B, 1, L, 1), kv[:, :, 1].transpose(1, 2), 0.0).reshape(B * Hk, L, hd)
    u = torch.matmul(qb, kb.contiguous()).view(B, Hk, n, H // Hk, L) * (1 / math.sqrt(hd))
    u = u - s["incl"].view(1, Hk, 1, H // Hk, 1) * (i - j).float()
    u = torch.where(vis, u, -math.inf)
    maior = u.amax(-1, keepdim=True)
    p = torch.exp(u - torch.where(maior == -math.inf, 0.0, maior))
    soma = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B * Hk, -1, L), vb).view(B, Hk, n, H // Hk, hd) / torch.where(soma == 0, 1.0, soma)
    y = torch.zeros(M, H * hd, device=DEV)
    y[linha[tem]] = o.permute(0, 2, 1, 3, 4).reshape(B, n, H * hd)[tem]
    if c["saida"] == "bloco":
        return _vale(*_bloco(y, blk), blk).to(torch.bfloat16)
    return y.to(torch.bfloat16) if c["saida"] == "bf16" else y


def _grava(c, s):
    """Every row's keys and values into the slot of its position; rows behind the last sequence write nothing."""
    H, Hk, hd, blk, pag = c["H"], c["Hk"], c["hd"], c["blk"], c["pag"]
    gs, G = _grupos(c)
    m, E = s["cache"]
    b, pos = _linhas(s)
    r = (b >= 0).nonzero().squeeze(1)
    b, pos = b[r], pos[r]
    pg, vaga = s["tabela"][b, pos // pag].long(), pos % pag
    col = torch.arange((H + 2 * Hk) * hd // gs, device=DEV) * gs // blk
    e = s["qkv"][1][:, col].view(-1, H + 2 * Hk, G)[r, H:].view(-1, 2, Hk, G)
    m[pg, c["camadas"] - 1, :, :, vaga] = s["qkv"][0].view(-1, H + 2 * Hk, hd)[r, H:].reshape(-1, 2, Hk, hd)
    E[pg, c["camadas"] - 1, :, :, vaga] = e
    return m, E


def _copia(c, s):
    m, E = s["cache"]
    de, para = torch.tensor(s["pares"], device=DEV).t()
    m[para], E[para] = m[de], E[de]
    return m, E


def _desempacota(W, N, K, blk):
    """The signed 4-bit weights [N, K] and scales [N, K / blk] of the packed layout."""
    m, esc, _ = W
    Nt, Kt = m.shape[:2]
    t = m.view(Nt, Kt, 4, 16, 4, 4)
    t = torch.stack([t & 15, t >> 4], -1).to(torch.int8)
    t = torch.where(t > 7, t - 16, t).permute(0, 3, 1, 4, 2, 6, 5).reshape(Nt * 16, Kt * 128)
    return t[:N, :K], esc.permute(0, 2, 1, 3).reshape(Nt * 16, -1)[:N, :K // blk]


def _produto4(c, s):
    """acc = sum over groups of rnd(p esc 2^(ea - RA) 2^-g), half to even, e = RA + R + g with g = log2(blk) - 4: p the
    exact dot product of a group, RA the largest exponent of x's row. p < 2^24 is exact in float32, the rest in float64."""
    M, N, K, blk = c["M"], c["N"], c["K"], c["blk"]
    x, ex = s["x"]
    w, esc = _desempacota(s["W"], N, K, blk)
    nb, g = K // blk, int(math.log2(blk)) - 4
    RA = ex.long().amax(1, keepdim=True)
    p = torch.matmul(x.view(M, nb, blk).transpose(0, 1).float().contiguous(), w.view(N, nb, blk).permute(1, 2, 0).float().contiguous())
    k = torch.exp2((ex.long() - RA - g).double()).t().unsqueeze(2) * esc.t().double().unsqueeze(1)      # [nb, M, N]
    acc = torch.round(p.double() * k).sum(0)
    return acc.to(torch.int32), (RA + s["W"][2].long() + g).to(torch.int16)


def _gemv4(c, s):
    acc, e = _produto4(c, s)
    if c["modo"] == "cru":
        return acc, e
    blk = c["blk"]
    y = _vale(*_bloco(acc.double() * torch.exp2(e.double()), blk), blk)
    if c["modo"] == "soma":
        y = y.double() + _vale(*s["res"], blk).double()     # aligned to 21 bits below the larger exponent: exact but for
        return _vale(*_bloco(y, blk), blk).to(torch.bfloat16)  # what lies 2^-22 of the block's largest value lower
    return _vale(*_bloco(y.clamp(min=0).double() ** 2, blk), blk).to(torch.bfloat16)


# ------------------------------------------------------------------------------------------------ work
def work(case):
    c = case
    if c["tipo"] == "gemv4":
        M, N, K, blk = c["M"], c["N"], c["K"], c["blk"]
        saida = 6 if c["modo"] == "cru" else 3 + 2 / blk if c["modo"] == "soma" else 2 + 1 / blk
        return dict(bytes=N * K * (0.5 + 2 / blk) + 2 * N + M * K * (1 + 1 / blk) + saida * M * N, flops=2 * M * N * K)
    gs, G = _grupos(c)
    token = 2 * c["Hk"] * (c["hd"] + G)                                # of a token's keys and values, in bytes
    if c["tipo"] == "copia":
        return dict(bytes=2 * c["pares"] * c["pag"] * c["camadas"] * token, flops=0)
    comp, novos = _comprimentos(c)
    if c["tipo"] == "grava":
        return dict(bytes=2 * sum(novos) * token, flops=0)
    lidos = pares = 0
    for L, n in zip(comp, novos):
        vis = lambda i, W=c["janela"], S=c["sumid"]: i + 1 if not W or i + 1 <= W else W + min(S, i + 1 - W)
        pares += sum(vis(i) for i in range(L - n, L))
        lidos += min(L, vis(L - 1) + n - 1) if n else 0
    D = c["H"] * c["hd"]
    return dict(bytes=lidos * token + sum(novos) * D * (1 + 1 / c["blk"] + dict(bf16=2, f32=4, bloco=3)[c["saida"]]), flops=4 * pares * D)


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["tipo"] == "atencao":
        return _exato_atencao(c, s)
    return _exato_gemv4(c, s) if c["tipo"] == "gemv4" else None       # the page operators compute no numbers


def _exato_atencao(c, s):
    """Row by row of a sequence's pages, one head's keys at a time where there are many rows."""
    H, Hk, hd, pag, Gq = c["H"], c["Hk"], c["hd"], c["pag"], c["H"] // c["Hk"]
    (qm, qE), (cm, cE), (gs, G) = s["qkv"], s["cache"], _grupos(c)
    escala = torch.pow(2.0, qE.double()).repeat_interleave(c["blk"], 1)
    q = (qm.double() * escala)[:, :H * hd].reshape(-1, H, hd)
    y = torch.zeros(qm.shape[0], H, hd, dtype=torch.float64, device=DEV)
    ini, comp, incl = s["ini"].tolist(), s["comp"].tolist(), s["incl"].double()
    for b in range(c["B"]):
        L, n = comp[b], ini[b + 1] - ini[b]
        if n == 0:
            continue
        i = torch.arange(L - n, L, device=DEV).unsqueeze(1)
        j = torch.arange(L, device=DEV)
        ve = j <= i
        if c["janela"]:
            ve &= (i - j < c["janela"]) | (j < c["sumid"])
        uso = ve.any(0).nonzero().squeeze(1)                           # the tokens that any row sees
        pg, vaga = s["tabela"][b].long()[uso // pag], uso % pag
        tk = cm[pg, c["camadas"] - 1, :, :, vaga].double() * torch.pow(2.0, cE[pg, c["camadas"] - 1, :, :, vaga].double()).repeat_interleave(gs, -1)
        ve, dist = ve[:, uso], (i - uso).double()
        for h in range(H):
            k, v = tk[:, 0, h // Gq], tk[:, 1, h // Gq]
            u = torch.mm(q[ini[b]:ini[b + 1], h], k.t()) / math.sqrt(hd) - incl[h] * dist
            u = u.masked_fill(~ve, -math.inf)
            p = torch.exp(u - u.max(1, keepdim=True).values)
            y[ini[b]:ini[b + 1], h] = torch.mm(p, v) / p.sum(1, keepdim=True)
    y = y.view(-1, H * hd)
    if c["saida"] != "bloco":
        return y
    m, E = _bloco(y, c["blk"])
    return m.double() * torch.pow(2.0, E.double()).repeat_interleave(c["blk"], 1)


def _exato_gemv4(c, s):
    """In 64-bit integers: a scale is s 2^-t with s of 8 bits; rnd is a shift with the remainder's half compared."""
    M, N, K, blk = c["M"], c["N"], c["K"], c["blk"]
    w, esc = _desempacota(s["W"], N, K, blk)
    f, t = torch.frexp(esc.double())
    s8, t = (f * 256).long(), 8 - t.long()
    (x, ex), nb = s["x"], K // blk
    ex, g = ex.long(), (1 if blk == 32 else 3)
    RA = ex.max(1).values
    acc = torch.zeros(M, N, dtype=torch.int64, device=DEV)
    xi, wi = x.view(M, nb, blk), w.view(N, nb, blk)
    for b in range(nb):
        p = torch.mm(xi[:, b].double(), wi[:, b].double().t()).long() * s8[:, b]
        sh = ((RA - ex[:, b]).unsqueeze(1) + t[:, b] + g).clamp(max=60)
        piso = p >> sh
        resto, meio = p - (piso << sh), torch.ones_like(sh) << (sh - 1).clamp(min=0)
        acc += torch.where(sh > 0, piso + ((resto > meio) | ((resto == meio) & (piso % 2 == 1))).long(), p << (-sh).clamp(min=0))
    e = RA.unsqueeze(1) + s["W"][2].long() + g
    if c["modo"] == "cru":
        return acc.to(torch.int32), e.to(torch.int16)
    val = lambda m, E: m.double() * torch.pow(2.0, E.double()).repeat_interleave(blk, 1)
    h = val(*_bloco(acc.double() * torch.pow(2.0, e.double()), blk))
    z = h + val(*s["res"]) if c["modo"] == "soma" else torch.relu(h) ** 2
    return val(*_bloco(z, blk))
