"""Performance cases of the 8-bit paged KV cache: its writes and reads, and the attention over it.

Four operators, each over the range a serving engine meets it in:

* ``store``   a chunk's (or a decode step's) K/V quantised into its pages, and those tokens read back;
* ``read``    the tokens of whole sequences read back from their pages in 16 bits;
* ``decode``  one layer's attention of a decode batch, one query token per sequence;
* ``chunk``   one layer's causal attention of packed chunk queries behind their prefixes.

The cache of a layer is codes [pages, 16, heads, dim] for K and for V, int8 or float8_e4m3fn, with one
power-of-two exponent byte for every 32 dims of a token's head, [pages, heads, ceil(dim / 32), 16] uint8.
With A the largest magnitude of such a block and M the format's largest code (127 or 448), the exponent
is the smallest e with M * 2^e >= A, kept within [-24, 9] (int8) or [-15, 7] (fp8), the byte e + 127, and
a code the value x * 2^-e rounded to the nearest, ties to even, magnitudes above M taken as M. A value
reads back as code * 2^e, which fp16 and bf16 hold exactly. A block with a NaN or an infinity has the
byte 255 and reads as NaN.

A case is a dict of plain values; lengths follow from its ``mix``, values and page placements from
``prepare``'s seed. Head shapes are those of ``perf/cases.py``.
"""
import math

import numpy as np
import torch

PAGE = 16
BLOCK = 32
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
# largest code, lowest and highest exponent, and the code that a block of NaN holds
FORMATS = {"int8": (127.0, -24, 9, 0), "fp8": (448.0, -15, 7, 0x7F)}

own = False


# ------------------------------------------------------------------------------------- cases
def listed():
    llama = dict(kv_heads=8, n_rep=4, dim=128)
    qwen = dict(kv_heads=4, n_rep=7, dim=128)
    small = dict(kv_heads=8, n_rep=4, dim=64)
    return [
        # A decode step's new tokens into the cache and back: the smallest call, where latency counts.
        dict(name="store_step", kind="store", fmt="int8", dtype="fp16", batch=8, prefix_lo=2049, prefix_hi=2600,
             chunk_lo=1, chunk_hi=1, mix=1, **qwen),
        # A prefill chunk of four sequences behind long prefixes.
        dict(name="store_chunk", kind="store", fmt="fp8", dtype="bf16", batch=4, prefix_lo=16384, prefix_hi=16384,
             chunk_lo=2048, chunk_hi=2048, mix=2, **llama),
        # A group of short prompts of ragged lengths, 64-dim heads.
        dict(name="store_prompts", kind="store", fmt="int8", dtype="fp16", batch=12, prefix_lo=0, prefix_hi=0,
             chunk_lo=16, chunk_hi=700, mix=3, **small),
        # Whole sequences read back for a step that takes 16-bit rows (scoring, moving to a 16-bit pool).
        dict(name="read_long", kind="read", fmt="int8", dtype="bf16", batch=4, lens="uniform", lo=16384, hi=32768,
             mix=4, **llama),
        dict(name="read_short", kind="read", fmt="fp8", dtype="fp16", batch=6, lens="uniform", lo=17, hi=900, mix=5,
             **qwen),
        # The smallest decode call: four chats of a few hundred to two thousand tokens.
        dict(name="decode_tiny", kind="decode", fmt="int8", dtype="fp16", batch=4, lens="uniform", lo=256, hi=2048,
             mix=6, **llama),
        # 16 sequences at 32K context, the most bytes a decode call reads here.
        dict(name="decode_long", kind="decode", fmt="fp8", dtype="bf16", batch=16, lens="uniform", lo=32768, hi=32768,
             mix=7, **llama),
        # A mixed batch: 64 sequences, lognormal lengths with a median near 2000.
        dict(name="decode_ragged", kind="decode", fmt="int8", dtype="bf16", batch=64, lens="lognormal", lo=128,
             hi=32768, mix=8, **llama),
        # Chunked prefill at long prefixes, the largest attention call.
        dict(name="chunk_long", kind="chunk", fmt="int8", dtype="bf16", batch=4, prefix_lo=16384, prefix_hi=16384,
             chunk_lo=2048, chunk_hi=2048, mix=9, **llama),
        # The online scheduler's chunk: four sequences, 512 tokens each, somewhere in their prompts.
        dict(name="chunk_mid", kind="chunk", fmt="fp8", dtype="fp16", batch=4, prefix_lo=500, prefix_hi=8000,
             chunk_lo=512, chunk_hi=512, mix=10, **qwen),
        # A few drafted tokens for each of sixteen long sequences, to be verified in one call.
        dict(name="chunk_drafts", kind="chunk", fmt="fp8", dtype="bf16", batch=16, prefix_lo=4000, prefix_hi=32000,
             chunk_lo=1, chunk_hi=8, mix=11, **llama),
        # A group of short prompts prefilled at once, no prefix, 64-dim heads.
        dict(name="chunk_prompts", kind="chunk", fmt="int8", dtype="fp16", batch=12, prefix_lo=0, prefix_hi=0,
             chunk_lo=16, chunk_hi=700, mix=12, **small),
    ]


# No drawn case moves more bytes or computes more than the largest listed one of its kind.
MAX_BYTES = {"store": 3.0e8, "read": 4.0e8, "decode": 1.1e9, "chunk": 4.0e8}
MAX_FLOPS = 2.3e12
MAX_SCORES = 4.9e9  # of the plain form, which holds a chunk's scores


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_once(rng):
    kind = rng.choice(["store", "read", "decode", "decode", "chunk", "chunk"])
    heads, n_rep = rng.choice([(8, 4), (8, 4), (4, 7), (4, 7), (1, 4), (2, 4), (1, 7), (2, 7), (8, 1), (4, 8)])
    case = dict(kind=kind, fmt=rng.choice(["int8", "fp8"]), dtype=rng.choice(["bf16", "fp16"]),
                mix=rng.randrange(1 << 30), kv_heads=heads, n_rep=n_rep, dim=rng.choice([128, 128, 64]))
    if kind in ("read", "decode"):
        case.update(batch=_log_int(rng, 1, 64), lens=rng.choice(["uniform", "lognormal"]))
        case["lo"] = _log_int(rng, 1, 8192)
        case["hi"] = max(case["lo"], _log_int(rng, 17, 32768))
    else:
        case["batch"] = _log_int(rng, 1, 32)
        case["prefix_lo"] = 0 if rng.random() < 0.3 else _log_int(rng, 1, 16384)
        case["prefix_hi"] = 0 if case["prefix_lo"] == 0 else max(case["prefix_lo"], _log_int(rng, 16, 32768))
        case["chunk_lo"] = _log_int(rng, 1, 1024)
        case["chunk_hi"] = max(case["chunk_lo"], _log_int(rng, 1, 2048))
    return case


def draw(rng):
    while True:
        case = _draw_once(rng)
        w = work(case)
        if w["bytes"] > MAX_BYTES[case["kind"]] or w["flops"] > MAX_FLOPS:
            continue
        pre, chunk = _split(case)
        longest = max(p + c for p, c in zip(pre, chunk))
        queries = 1 if case["kind"] != "chunk" else max(chunk)
        if case["batch"] * case["kv_heads"] * case["n_rep"] * queries * longest <= MAX_SCORES and \
                case["batch"] * case["kv_heads"] * case["dim"] * longest <= 2.2e9:
            return case


# ------------------------------------------------------------------------------------ layouts
def _split(case):
    """(tokens before, tokens of the call) of each sequence."""
    rng = np.random.default_rng(case["mix"])
    n = case["batch"]
    if case["kind"] in ("read", "decode"):
        if case["lens"] == "uniform":
            lens = rng.integers(case["lo"], case["hi"], size=n, endpoint=True)
        else:
            raw = rng.lognormal(mean=math.log(math.sqrt(case["lo"] * case["hi"])), sigma=1.0, size=n)
            lens = np.clip(np.round(raw), case["lo"], case["hi"])
        if case["kind"] == "read":
            return [0] * n, [int(x) for x in lens]
        return [int(x) - 1 for x in lens], [1] * n
    pre = rng.integers(case["prefix_lo"], case["prefix_hi"], size=n, endpoint=True)
    chunk = rng.integers(case["chunk_lo"], case["chunk_hi"], size=n, endpoint=True)
    return [int(x) for x in pre], [int(x) for x in chunk]


def _pages(n_tokens):
    return -(-n_tokens // PAGE)


def work(case):
    pre, chunk = _split(case)
    H, R, D = case["kv_heads"], case["n_rep"], case["dim"]
    row16 = 2 * 2 * H * D  # a token's K and V in 16 bits
    row8 = 2 * H * (D + -(-D // BLOCK))
    small = 4 * case["batch"] * (2 + max(_pages(p + c) for p, c in zip(pre, chunk)))
    new, keys = sum(chunk), sum(p + c for p, c in zip(pre, chunk))
    if case["kind"] == "store":
        return {"bytes": new * 2 * (row16 + row8) + small, "flops": 0}
    if case["kind"] == "read":
        return {"bytes": new * (row16 + row8) + small, "flops": 0}
    pairs = sum(c * p + c * (c + 1) // 2 for p, c in zip(pre, chunk))
    return {"bytes": keys * row8 + 2 * 2 * new * H * R * D + small, "flops": 4 * H * R * D * pairs}


# ------------------------------------------------------------------------------ plain quantiser
def _pow2(e):
    """2^e in fp32 for integers e of [-126, 127], exactly."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantise(x, fmt):
    """Rows [..., heads, dim] -> (codes uint8 [..., heads, dim], exponent bytes uint8 [..., heads, blocks])."""
    top, lo, hi, nan_code = FORMATS[fmt]
    D = x.shape[-1]
    blocks = -(-D // BLOCK)
    y = torch.nn.functional.pad(x.float(), (0, blocks * BLOCK - D)).unflatten(-1, (blocks, BLOCK))
    largest = y.abs().amax(-1)
    bad = ~torch.isfinite(largest)
    # top * 2^e >= largest, decided on the fp32 numbers' own exponent and fraction
    fraction, power = torch.frexp(torch.where(bad, 0.0, largest))
    top_fraction, top_power = math.frexp(top)
    e = torch.where(largest == 0, lo, power - top_power + (fraction > top_fraction)).clamp(lo, hi)
    scaled = (y * _pow2(-e)[..., None]).clamp(-top, top)
    if fmt == "int8":
        codes = torch.where(bad[..., None], 0.0, scaled).round().to(torch.int8).view(torch.uint8)
    else:
        codes = torch.where(bad[..., None], 0.0, scaled).to(torch.float8_e4m3fn).view(torch.uint8)
    codes = torch.where(bad[..., None], nan_code, codes).flatten(-2)[..., :D]
    return codes.contiguous(), torch.where(bad, 255, e + 127).to(torch.uint8)


def _values(codes, exponents, fmt):
    """Codes uint8 [..., heads, dim] and exponent bytes [..., heads, blocks] -> fp32 values."""
    x = codes.view(torch.int8 if fmt == "int8" else torch.float8_e4m3fn).float()
    scale = torch.where(exponents == 255, math.nan, _pow2(exponents.to(torch.int32) - 127))
    return x * scale.repeat_interleave(BLOCK, -1)[..., :x.shape[-1]]


# ------------------------------------------------------------------------------------ prepare
def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt, fmt = DTYPES[case["dtype"]], case["fmt"]
    H, R, D, B = case["kv_heads"], case["n_rep"], case["dim"], case["batch"]
    pre, chunk = _split(case)
    counts = [_pages(p + c) for p, c in zip(pre, chunk)]
    pool = sum(counts) + max(8, sum(counts) // 10)  # a pool is never quite full
    perm = np.random.default_rng(seed).permutation(pool)
    table = np.zeros((B, max(counts)), dtype=np.int32)
    at = 0
    for row, n in zip(table, counts):
        row[:n] = perm[at:at + n]
        at += n
    # K channels differ in size, as a model's do: some are several times the others.
    size = torch.exp(torch.randn((H, D), generator=gen, device="cuda") * 0.5)
    state = dict(case=case, fmt=fmt, dtype=dt, total=sum(chunk), max_chunk=max(chunk), max_len=PAGE * max(counts),
                 scale=1.0 / math.sqrt(D), n_rep=R, table=torch.from_numpy(table).cuda())
    for name in ("k", "v"):
        codes = torch.empty((pool, PAGE, H, D), dtype=torch.uint8, device="cuda")
        exps = torch.empty((pool, H, -(-D // BLOCK), PAGE), dtype=torch.uint8, device="cuda")
        step = max(1, (1 << 26) // (PAGE * H * D))
        for lo in range(0, pool, step):
            n = min(step, pool - lo)
            x = torch.randn((n, PAGE, H, D), generator=gen, device="cuda")
            c, e = _quantise((x * size if name == "k" else x).to(dt), fmt)
            codes[lo:lo + n] = c
            exps[lo:lo + n] = e.permute(0, 2, 3, 1)
        state[name + "_codes"], state[name + "_scale"] = codes, exps
    cu = np.concatenate([[0], np.cumsum(chunk)])
    state["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
    state["before"] = torch.tensor(pre, dtype=torch.int32, device="cuda")
    state["lens"] = torch.tensor([p + c for p, c in zip(pre, chunk)], dtype=torch.int32, device="cuda")
    if case["kind"] == "store":
        state["k_new"] = (torch.randn((sum(chunk), H, D), generator=gen, device="cuda") * size).to(dt)
        state["v_new"] = torch.randn((sum(chunk), H, D), generator=gen, device="cuda").to(dt)
    elif case["kind"] != "read":
        state["q"] = torch.randn((sum(chunk), H * R, D), generator=gen, device="cuda").to(dt)
    return state


# ---------------------------------------------------------------------------------------- run
def _slots(state):
    """Page and slot in it of each packed row of the call."""
    cu = state["cu"].long()
    seq = torch.repeat_interleave(torch.arange(len(cu) - 1, device=cu.device), cu.diff(), output_size=state["total"])
    at = torch.arange(state["total"], device=cu.device) - cu[seq] + state["before"].long()[seq]
    return seq, at, state["table"][seq, at // PAGE].long(), at % PAGE


def _gathered(state, name):
    """Every page of the batch's table as fp32 [batch, heads, tokens, dim]."""
    table = state["table"].long()
    x = _values(state[name + "_codes"][table], state[name + "_scale"][table].permute(0, 1, 4, 2, 3), state["fmt"])
    return x.flatten(1, 2).transpose(1, 2)


def _attend(q, k, v, seen, scale):
    """softmax(scale q k^T) v over the keys t < seen of each row: q [batch, heads, rows, dim], seen [batch, 1, rows]."""
    s = torch.matmul(q * scale, k.transpose(-1, -2))
    s.masked_fill_(torch.arange(k.shape[-2], device=q.device) >= seen[..., None], -math.inf)
    s -= s.amax(-1, keepdim=True)
    s.exp_()
    return torch.matmul(s, v) / s.sum(-1, keepdim=True)


def _plain(state):
    kind, fmt, dt = state["case"]["kind"], state["fmt"], state["dtype"]
    if kind in ("store", "read"):
        _, _, page, slot = _slots(state)
        if kind == "store":
            for name in ("k", "v"):
                codes, exps = _quantise(state[name + "_new"], fmt)
                state[name + "_codes"][page, slot] = codes
                state[name + "_scale"].permute(0, 3, 1, 2)[page, slot] = exps
        rows = [(state[n + "_codes"][page, slot], state[n + "_scale"].permute(0, 3, 1, 2)[page, slot]) for n in "kv"]
        return [_values(codes, exps, fmt).to(dt) for codes, exps in rows]
    H, R, D = (state["case"][x] for x in ("kv_heads", "n_rep", "dim"))
    q = state["q"].float()
    if kind == "decode":
        rows = q.unflatten(1, (H, R))
        seen = state["lens"][:, None, None].expand(-1, 1, R)
        out = _attend(rows, _gathered(state, "k"), _gathered(state, "v"), seen, state["scale"])
        return out.flatten(1, 2).to(dt)
    # packed rows -> [batch, heads, n_rep * longest chunk, dim], and back
    seq, at, _, _ = _slots(state)
    i = at - state["before"].long()[seq]
    B, C = state["case"]["batch"], state["max_chunk"]
    padded = q.new_zeros((B, C, H * R, D))
    padded[seq, i] = q
    rows = padded.unflatten(2, (H, R)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    seen = (state["before"][:, None] + 1 + torch.arange(C, device=q.device)).repeat(1, R)[:, None]
    out = _attend(rows, _gathered(state, "k"), _gathered(state, "v"), seen, state["scale"])
    out = out.unflatten(2, (R, C)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    return out[seq, i].to(dt)


def _layer(state):
    from unifiedkv_amd import quant_kv

    of = torch.int8 if state["fmt"] == "int8" else torch.float8_e4m3fn
    return quant_kv.QuantLayer(state["k_codes"].view(of), state["v_codes"].view(of), state["k_scale"], state["v_scale"])


def _framework(state):
    from unifiedkv_amd import quant_kv

    kind, layer = state["case"]["kind"], _layer(state)
    if kind in ("store", "read"):
        if kind == "store" and state["max_chunk"] == 1:  # a decode step appends
            quant_kv.append_kv(layer, state["k_new"], state["v_new"], state["table"], state["before"])
        elif kind == "store":
            quant_kv.write_chunk_kv(layer, state["k_new"], state["v_new"], state["table"], state["cu"], state["lens"],
                                    max_chunk=state["max_chunk"])
        return list(quant_kv.read_kv(layer, state["table"], state["cu"], state["lens"], dtype=state["dtype"],
                                     max_chunk=state["max_chunk"], total=state["total"]))
    if kind == "decode":
        return quant_kv.decode_attention(state["q"], layer, state["table"], state["lens"],
                                         softmax_scale=state["scale"], n_rep=state["n_rep"])
    return quant_kv.prefill_attention(state["q"], layer, state["table"], state["cu"], state["lens"],
                                      softmax_scale=state["scale"], n_rep=state["n_rep"], max_chunk=state["max_chunk"])


def run(state):
    if own:
        return _framework(state)
    return _plain(state)


# -------------------------------------------------------------------------------------- exact
def _exact_tables(fmt):
    """The fp64 value of each of the 256 codes and of each of the 256 exponent bytes, from the formats' definitions."""
    code = np.arange(256, dtype=np.uint8)
    if fmt == "int8":
        x = code.view(np.int8).astype(np.float64)
    else:  # sign, four exponent bits biased by 7, three fraction bits; all ones is NaN
        e, m = ((code >> 3) & 15).astype(np.float64), (code & 7) / 8.0
        x = np.where(e == 0, m * 2.0 ** -6, (1 + m) * 2.0 ** (e - 7)) * np.where(code >> 7, -1.0, 1.0)
        x[[0x7F, 0xFF]] = np.nan
    scale = 2.0 ** (np.arange(256) - 127.0)
    scale[255] = np.nan
    return torch.from_numpy(x).cuda(), torch.from_numpy(scale).cuda()


def _exact_rounded(x, fmt):
    """What rows fp64 [tokens, heads, dim] read back as: each block's exponent, then each value to the nearest step."""
    top, lo, hi, _ = FORMATS[fmt]
    out = np.empty_like(x)
    for d in range(0, x.shape[-1], BLOCK):
        y = x[..., d:d + BLOCK]
        largest = np.abs(y).max(-1, keepdims=True)
        e = np.full(largest.shape, lo, dtype=np.float64)
        for step in range(lo, hi):
            e = np.where(top * 2.0 ** step < largest, step + 1.0, e)
        z = np.clip(y / 2.0 ** e, -top, top)
        if fmt == "int8":
            step = np.ones_like(z)
        else:  # eight steps a binade down to 2^-6, 2^-9 below
            step = 2.0 ** (np.maximum(np.floor(np.log2(np.maximum(np.abs(z), 2.0 ** -9))), -6) - 3)
        z = np.round(z / step) * step
        out[..., d:d + BLOCK] = np.where(np.isfinite(largest), z * 2.0 ** e, np.nan)
    return out


def exact(case, seed):
    state = prepare(case, seed)
    pre, chunk = _split(case)
    H, R, D, fmt = case["kv_heads"], case["n_rep"], case["dim"], case["fmt"]
    if case["kind"] == "store":
        return [_exact_rounded(state[n].double().cpu().numpy(), fmt) for n in ("k_new", "v_new")]
    value, power = _exact_tables(fmt)

    def head(name, b, h):
        """The tokens of one head of one sequence, fp64 [tokens, dim]."""
        n = pre[b] + chunk[b]
        ids = state["table"][b, :_pages(n)].long()
        codes = value[state[name + "_codes"][ids, :, h].long()].reshape(-1, D)
        scales = power[state[name + "_scale"][ids, h].long()].permute(0, 2, 1).reshape(len(codes), -1)
        return (codes * torch.repeat_interleave(scales, BLOCK, -1)[:, :D])[:n]

    if case["kind"] == "read":
        return [torch.cat([torch.stack([head(n, b, h) for h in range(H)], 1) for b in range(len(chunk))])
                for n in ("k", "v")]
    q = state["q"].double()
    out, row = torch.empty_like(q), 0
    for b, (p, c) in enumerate(zip(pre, chunk)):
        unseen = torch.arange(p + c, device="cuda")[None] > (p + torch.arange(c, device="cuda"))[:, None]
        for h in range(H):
            k, v = head("k", b, h), head("v", b, h)
            for r in range(h * R, (h + 1) * R):
                s = (q[row:row + c, r] @ k.T / math.sqrt(D)).masked_fill_(unseen, -math.inf)
                out[row:row + c, r] = torch.softmax(s, -1) @ v
        row += c
    return out
