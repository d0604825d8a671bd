"""Operators of a layer in 8-bit integers whose batch shares prompts, as cases to time and compare.

Three kinds, each through the public entry points of ferret_amd.ops:

  quant   bf16 rows to int8 codes with one fp32 scale per token.
  gemm    the product of int8 codes with a scale per token and per output
          channel, the residual's addition where one is given.
  shared  latent attention over the paged cache of a batch whose sequences share
          prefixes (a system prompt, or each prompt of several samples): keys of
          the prefix that every token of its sequences sees, then the
          sequence's own, new tokens included.

A token's codes are q = round(127 x / a) with a = max |x| and the scale a / 127, ties
to even; rows below 2^-100 take a = 2^-100.  A cached row is as in the framework's
latent cache: 512 latents and 64 rotary values, 576 bf16, or 640 bytes (512 e4m3 codes,
the rotary values in bf16) with four exponent bytes in a tensor of their own (byte b:
2^(b - 127)).

Sizes are those of the framework's projections and attention heads: 16 heads on a
rank of 8, 128 on one GPU.
"""
import math

import torch

own = False

DEV = "cuda"
FP8 = torch.float8_e4m3fn
LATENT, ROTARY = 512, 64
ROW, ROW8 = LATENT + ROTARY, LATENT + 2 * ROTARY
SCALE = 192 ** -0.5
MIN_BYTE = 16  # the smallest exponent byte: every code times its scale is a normal bf16 value
LEAST = 2.0 ** -100  # rows with a smaller largest value are quantised as if it were this


def listed():
    return [
        # The activations of a decode step of 32 sequences: latency.
        {"name": "quant_decode_M32", "kind": "quant", "M": 32, "K": 4096, "wide": 0},
        # The activations of a prefill batch: memory bandwidth.
        {"name": "quant_prefill_M8192", "kind": "quant", "M": 8192, "K": 7168, "wide": 0},
        # One token of one sequence through the gate-up projection: the weights' bytes.
        {"name": "gemm_gateup_M1", "kind": "gemm", "M": 1, "N": 24576, "K": 4096, "residual": False},
        # The down projection of a decode step of 16 sequences, its residual added.
        {"name": "gemm_down_M16_res", "kind": "gemm", "M": 16, "N": 4096, "K": 12288, "residual": True},
        # One rank's attention output projection for a ragged decode batch.
        {"name": "gemm_oproj_M100", "kind": "gemm", "M": 100, "N": 7168, "K": 2048, "residual": False},
        # The QKV projection of a chunk of a ragged prompt.
        {"name": "gemm_qkv_M1000", "kind": "gemm", "M": 1000, "N": 6144, "K": 4096, "residual": False},
        # A full prefill batch through a dense projection: matrix products.
        {"name": "gemm_dense_M4096", "kind": "gemm", "M": 4096, "N": 4096, "K": 7168, "residual": False},
        # A decode step of a few sequences behind a short system prompt: latency.
        {"name": "shared_small_B4", "kind": "shared", "H": 16, "G": 1, "B": 4, "prefix_lo": 500, "prefix_hi": 500,
         "lo": 20, "hi": 150, "new_lo": 1, "new_hi": 1, "page": 64, "e4m3": True},
        # A decode step of 64 sequences behind one system prompt, on one rank's 16 heads.
        {"name": "shared_decode_H16_B64", "kind": "shared", "H": 16, "G": 1, "B": 64, "prefix_lo": 8192,
         "prefix_hi": 8192, "lo": 100, "hi": 1200, "new_lo": 1, "new_hi": 1, "page": 64, "e4m3": True},
        # Eight prompts, eight samples of each.
        {"name": "shared_samples_H16_G8", "kind": "shared", "H": 16, "G": 8, "B": 64, "prefix_lo": 600,
         "prefix_hi": 3500, "lo": 10, "hi": 500, "new_lo": 1, "new_hi": 1, "page": 64, "e4m3": False},
        # A decode step with all 128 heads on one GPU behind one document.
        {"name": "shared_decode_H128_B32", "kind": "shared", "H": 128, "G": 1, "B": 32, "prefix_lo": 6001,
         "prefix_hi": 6001, "lo": 50, "hi": 800, "new_lo": 1, "new_hi": 1, "page": 64, "e4m3": False},
        # Questions of several users about one document: chunks of new tokens behind it.
        {"name": "shared_chunk_H16_B5", "kind": "shared", "H": 16, "G": 1, "B": 5, "prefix_lo": 5000,
         "prefix_hi": 5000, "lo": 100, "hi": 400, "new_lo": 60, "new_hi": 300, "page": 64, "e4m3": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["quant", "gemm", "gemm", "gemm", "shared", "shared", "shared"])
    if kind == "quant":
        K = 16 * _log_int(rng, 16, 768)
        wide = K + 8 * rng.randint(1, 100) if rng.random() < 0.3 else 0
        return {"kind": kind, "M": _log_int(rng, 1, 8192 * 7168 // max(K, 7168)), "K": K, "wide": wide}
    if kind == "gemm":
        M = _log_int(rng, 1, 8192)
        if rng.random() < 0.5:
            N, K = rng.choice([(6144, 4096), (4096, 4096), (24576, 4096), (4096, 12288), (4096, 7168), (7168, 2048),
                               (4096, 512)])
        else:
            N, K = 8 * _log_int(rng, 64, 2048), 16 * _log_int(rng, 16, 768)
        M = max(1, min(M, 4096 * 4096 * 7168 // (N * K)))
        return {"kind": kind, "M": M, "N": N, "K": K, "residual": rng.random() < 0.4}
    H = rng.choice([8, 16, 16, 32, 64, 128])
    G = rng.choice([1, 1, 1, 2, _log_int(rng, 2, 12)])
    B = G * _log_int(rng, 1, 96 // G) + rng.randint(0, G - 1)
    new = rng.choice([1, 1, 2, _log_int(rng, 3, 200)])
    if new > 2:
        B = max(G, min(B, 600 // new))
    tokens = B * new * H
    prefix = _log_int(rng, 64, max(65, min(32768, 70_000_000 // tokens, 120_000 // G)))
    hi = max(new, _log_int(rng, 16, max(17, min(4000, 60_000 // B, 20_000_000 // tokens))))
    return {"kind": kind, "H": H, "G": G, "B": B, "prefix_lo": rng.randint(max(1, prefix // 6), prefix),
            "prefix_hi": prefix, "lo": rng.randint(max(1, hi // 8), hi), "hi": hi, "new_lo": max(1, new // 3),
            "new_hi": new, "page": rng.choice([16, 32, 64, 128]), "e4m3": rng.random() < 0.5}


# ---- the ragged batch of a case: known from the case alone ------------------------------------------------------

def _spread(lo, hi, n):
    """n whole numbers from lo to hi, both among them where n > 1, in a mixed order."""
    if n == 1:
        return [hi]
    at = sorted(range(n), key=lambda i: (i * 0.6180339887498949) % 1.0)
    return [lo + (hi - lo) * k // (n - 1) for k in at]


def _starts(counts):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return at


def _batch(case):
    """(prefix lengths, sequences of each prefix, own lengths, new tokens of the sequences)."""
    G, B = case["G"], case["B"]
    prefix = _spread(case["prefix_lo"], case["prefix_hi"], G)
    members = [B // G + (1 if g < B % G else 0) for g in range(G)]
    lens = _spread(case["lo"], case["hi"], B)
    new = _spread(case["new_lo"], case["new_hi"], B)[::-1]
    return prefix, members, lens, [min(a, b) for a, b in zip(new, lens)]


def _tokens_of(members, new):
    """New tokens of each prefix's sequences."""
    at = _starts(members)
    return [sum(new[a:b]) for a, b in zip(at, at[1:])]


def work(case):
    if case["kind"] == "quant":
        return {"bytes": case["M"] * (3 * case["K"] + 4), "flops": 3 * case["M"] * case["K"]}
    if case["kind"] == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": (M + N) * (K + 4) + 2 * M * N * (2 if case["residual"] else 1), "flops": 2 * M * N * K}
    prefix, members, lens, new = _batch(case)
    row = (ROW8 + 4) if case["e4m3"] else 2 * ROW
    pairs = sum(n * (length - n) + n * (n + 1) // 2 for length, n in zip(lens, new))
    pairs += sum(p * t for p, t in zip(prefix, _tokens_of(members, new)))
    return {"bytes": (sum(prefix) + sum(lens)) * row + sum(new) * case["H"] * 2 * (ROW + LATENT),
            "flops": 2 * pairs * case["H"] * (ROW + LATENT)}


# ---- inputs -----------------------------------------------------------------------------------------------------

def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV).to(torch.bfloat16)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _activations(g, M, K):
    """Hidden states: a few channels far larger than the others, tokens of different size."""
    gain = torch.exp(0.6 * torch.randn(K, generator=g, device=DEV)).clamp(max=8)
    size = torch.exp(torch.randn((M, 1), generator=g, device=DEV))
    return (torch.randn((M, K), generator=g, device=DEV) * gain * size).to(torch.bfloat16)


def _codes(x):
    """Any rows to int8 codes and scales, as a program quantises its weights at load."""
    x = x.float()
    a = x.abs().amax(-1).clamp(min=LEAST)
    return torch.round(x * 127 / a[:, None]).to(torch.int8), a / 127


def _latents(g, rows):
    """Normed latents: unit variance, a few channels with larger weights."""
    gain = torch.exp(0.5 * torch.randn(LATENT, generator=g, device=DEV))
    return (torch.randn((rows, LATENT), generator=g, device=DEV) * gain.clamp(max=6)).to(torch.bfloat16)


def _quantize_latents(lat):
    """bf16 [n, 512] -> (e4m3 codes [n, 512], exponent bytes [n, 4]), both exact."""
    x = lat.float().view(-1, 4, 128)
    m, e = torch.frexp(x.abs().amax(-1))              # amax = m 2^e, 0.5 <= m < 1; 448 = 0.875 2^9
    byte = (e - 9 + (m > 0.875).to(e.dtype) + 127).clamp(min=MIN_BYTE)
    codes = torch.ldexp(x, (127 - byte).unsqueeze(-1)).to(FP8)
    return codes.view(-1, LATENT), byte.to(torch.uint8)


def _tables(case, groups, g):
    """Page tables of shuffled pages for several lists of lengths out of one pool, and the pool's pages."""
    page = case["page"]
    per = [[-(-n // page) for n in lens] for lens in groups]
    pages = sum(map(sum, per)) + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    tables, at = [], 0
    for counts in per:
        table = torch.zeros((len(counts), max(counts)), dtype=torch.int32, device=DEV)
        for b, n in enumerate(counts):
            table[b, :n] = order[at:at + n]
            at += n
        tables.append(table)
    return tables, pages


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": dict(case)}
    if case["kind"] == "quant":
        x = _activations(g, case["M"], case["wide"] or case["K"])
        s["x"] = x[:, x.shape[1] - case["K"]:] if case["wide"] else x
        return s
    if case["kind"] == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        s["a"], s["sa"] = _codes(_activations(g, M, K))
        s["b"], s["sb"] = _codes(0.02 * torch.randn((N, K), generator=g, device=DEV))
        s["residual"] = _randn(g, M, N) if case["residual"] else None
        return s
    prefix, members, lens, new = _batch(case)
    T, H = sum(new), case["H"]
    tokens = _tokens_of(members, new)
    s["prefix_lens"], s["lens"] = _ints(prefix), _ints(lens)
    s["cu_prefix"], s["cu_q"] = _ints(_starts(tokens)), _ints(_starts(new))
    s["longest_prefix"], s["longest"], s["most_tokens"], s["most"] = max(prefix), max(lens), max(tokens), max(new)
    (s["prefix_table"], s["table"]), pages = _tables(case, [prefix, lens], g)
    rows = pages * case["page"]
    if case["e4m3"]:
        codes, scales = _quantize_latents(_latents(g, rows))
        data = torch.cat([codes.view(torch.uint8), _randn(g, rows, ROTARY).view(torch.uint8)], -1)
        s["data"], s["scales"] = data.view(pages, -1, ROW8), scales.view(pages, -1, 4)
    else:
        s["data"], s["scales"] = torch.cat([_latents(g, rows), _randn(g, rows, ROTARY)], -1).view(pages, -1, ROW), None
    # the products with the key projection come head by head
    s["ql"], s["qr"] = _randn(g, H, T, LATENT).transpose(0, 1), _randn(g, T, H, ROTARY)
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------

def run(s):
    return (_own if own else _plain)(s)


def _own(s):
    from ferret_amd import ops
    kind = s["case"]["kind"]
    if kind == "quant":
        return ops.quant_act_int8(s["x"])
    if kind == "gemm":
        return ops.int8_gemm(s["a"], s["sa"], s["b"], s["sb"], s["residual"])
    return ops.latent_attention_shared(s["ql"], s["qr"], ops.LatentCache(s["data"], s["scales"]), s["prefix_table"],
                                       s["prefix_lens"], s["cu_prefix"], s["table"], s["lens"], s["cu_q"], scale=SCALE)


def _plain(s):
    kind = s["case"]["kind"]
    return {"quant": _plain_quant, "gemm": _plain_gemm, "shared": _plain_shared}[kind](s)


def _plain_quant(s):
    x = s["x"].float()
    a = x.abs().amax(-1).clamp(min=LEAST)
    return torch.round(x * 127 / a[:, None]).to(torch.int8), a / 127


def _plain_gemm(s):
    y = torch.matmul(s["a"].float(), s["b"].float().t()) * s["sa"][:, None] * s["sb"]
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(torch.bfloat16)


def _rows(s, table, longest, lens):
    """The cached rows of every line of a page table: [lines, longest, 576] in 32 bits; past a line's end its last."""
    page = s["case"]["page"]
    j = torch.arange(longest, device=DEV)[None].expand(lens.numel(), -1)
    j = torch.minimum(j, lens.long()[:, None] - 1)
    at = torch.gather(table.long(), 1, j // page) * page + j % page
    if s["scales"] is None:
        return s["data"].view(-1, ROW)[at].float()
    rows = s["data"].view(-1, ROW8)[at]
    lat = rows[..., :LATENT].view(FP8).float().view(*at.shape, 4, 128)
    lat = lat * torch.exp2(s["scales"].view(-1, 4)[at].float() - 127).unsqueeze(-1)
    return torch.cat([lat.view(*at.shape, LATENT), rows[..., LATENT:].contiguous().view(torch.bfloat16).float()], -1)


def _attend(q, starts, most, keys, limit):
    """Packed queries [T, H, 576], those of a line of keys padded to [lines, most]; `limit` [lines, most]: keys that a
    token sees.  Packed again: maxima [T, H], sums of exp, and the sums weighted by them [T, H, 512]."""
    H, m = q.shape[1], keys.shape[1]
    i = torch.arange(most, device=DEV)[None]
    at = (starts.long()[:-1, None] + i).clamp(max=q.shape[0] - 1)
    z = torch.matmul(q[at].view(len(at), most * H, ROW), keys.transpose(1, 2).contiguous()) * SCALE
    hidden = torch.arange(m, device=DEV)[None, None] >= limit[:, :, None]
    z = z.view(len(at), most, H, m).masked_fill(hidden[:, :, None], float("-inf"))
    top = z.amax(-1)
    p = torch.exp(z - top.unsqueeze(-1)).nan_to_num(0.0)
    o = torch.matmul(p.view(len(at), most * H, m), keys[..., :LATENT].contiguous()).view(len(at), most, H, LATENT)
    live = i < (starts[1:] - starts[:-1])[:, None]
    return top[live], p.sum(-1)[live], o[live]


def _plain_shared(s):
    q = torch.cat([s["ql"], s["qr"]], -1).float()
    keys = _rows(s, s["prefix_table"], s["longest_prefix"], s["prefix_lens"])
    limit = s["prefix_lens"][:, None].expand(-1, s["most_tokens"])
    m0, l0, o0 = _attend(q, s["cu_prefix"], s["most_tokens"], keys, limit)
    keys = _rows(s, s["table"], s["longest"], s["lens"])
    new = s["cu_q"][1:] - s["cu_q"][:-1]
    limit = (s["lens"] - new)[:, None] + 1 + torch.arange(s["most"], device=DEV)[None]
    m1, l1, o1 = _attend(q, s["cu_q"], s["most"], keys, torch.minimum(limit, s["lens"][:, None]))
    m = torch.maximum(m0, m1)
    w0, w1 = torch.exp(m0 - m), torch.exp(m1 - m)
    o = o0 * w0.unsqueeze(-1) + o1 * w1.unsqueeze(-1)
    return (o / (l0 * w0 + l1 * w1).unsqueeze(-1)).to(torch.bfloat16)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "quant":
        x = s["x"].double()
        a = torch.linalg.vector_norm(x, ord=float("inf"), dim=1).clamp(min=LEAST)
        return torch.round(x * 127 / a.unsqueeze(1)).to(torch.int8), a / 127
    if case["kind"] == "gemm":
        # whole numbers below 2^53: every sum is exact
        y = (s["a"].double() @ s["b"].double().T) * torch.outer(s["sa"].double(), s["sb"].double())
        return y if s["residual"] is None else y + s["residual"].double()
    prefix, members, lens, new = _batch(case)
    out, t, b = [], 0, 0
    for g, (length, count) in enumerate(zip(prefix, members)):
        first = _exact_rows(s, s["prefix_table"], g, length)
        for _ in range(count):
            n = new[b]
            keys = torch.cat([first, _exact_rows(s, s["table"], b, lens[b])])
            q = torch.cat([s["ql"][t:t + n], s["qr"][t:t + n]], -1).double()
            z = torch.einsum("thd,sd->ths", q, keys) * SCALE
            last = torch.arange(len(keys) - n, len(keys), device=DEV)
            z.masked_fill_((torch.arange(len(keys), device=DEV)[None] > last[:, None])[:, None], float("-inf"))
            out.append(torch.einsum("ths,sd->thd", torch.softmax(z, -1), keys[:, :LATENT]))
            t, b = t + n, b + 1
    return torch.cat(out)


def _exact_rows(s, table, line, n):
    page = s["case"]["page"]
    at = torch.tensor([int(p) * page + i for p in table[line].tolist() for i in range(page)][:n], device=DEV)
    if s["scales"] is None:
        return s["data"].reshape(-1, ROW)[at].double()
    rows = s["data"].reshape(-1, ROW8)[at]
    power = torch.pow(2.0, s["scales"].reshape(-1, 4)[at].double() - 127).repeat_interleave(128, 1)
    return torch.cat([rows[:, :LATENT].contiguous().view(FP8).double() * power,
                      rows[:, LATENT:].contiguous().view(torch.bfloat16).double()], -1)
