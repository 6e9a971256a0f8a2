"""The calls on an 8-bit paged cache that the speed of this library is measured on.

A server keeps keys and values in one byte an element: a code, int8 or e4m3, and for every key of a
key/value head one power of two, x - 127 of a byte x. Value = code * 2^(x - 127). A case is one call.
Fields:

  op      "append"   flash_attention_append_paged_q8: rotates the new tokens' queries and keys,
                     quantises keys and values and writes them to their pages
          "read"     flash_attention_read_paged_q8: the newest keys and values of every sequence
                     as numbers of `dtype`
          "decode"   flash_attention_decode_paged_q8: one query per sequence over the cache
          "forward"  flash_attention_forward_paged_q8: several new tokens' attention over it
  dtype   "float16", "bfloat16" or "float32": queries, new keys and values, outputs
  code    "int8" or "e4m3"
  B, H, Hkv, D, page   sequences, query heads, key/value heads, head_dim, keys per page
  new     most new tokens of a sequence (read: keys to read); sequence i of a batch has
          new (i + 1) / B of them, at least one, or all have `new` where `even`
  old     most keys that a sequence had before; old (B - i) / B of them
  causal  a token sees the keys up to its own ("forward")
  rotary, interleaved   rotated elements of a head, and whether a pair is (2i, 2i + 1) or
          (i, i + rotary / 2) ("append")

Codes and exponents are outputs as the cache holds them (int8 and e4m3 numbers, and whole numbers).
"""

import math
import os
import random
import sys

import torch

own = False

_TOP = {"int8": 127.0, "e4m3": 448.0}
# The largest exponent, by which the largest code stays finite in the type.
_MOST = {("int8", "float16"): 9, ("e4m3", "float16"): 7, ("int8", "bfloat16"): 121,
         ("e4m3", "bfloat16"): 119, ("int8", "float32"): 121, ("e4m3", "float32"): 119}
_LEAST = -100


def _case(op, dtype, code, B, H, Hkv, D, page, new=1, old=0, even=False, causal=True, rotary=0,
          interleaved=False, **name):
    return dict(name, op=op, dtype=dtype, code=code, B=B, H=H, Hkv=Hkv, D=D, page=page, new=new,
                old=old, even=even, causal=causal, rotary=rotary, interleaved=interleaved)


def listed():
    return [
        # One user's next token goes into the cache: the smallest call of a decode step.
        _case("append", "bfloat16", "e4m3", 1, 32, 8, 128, 16, old=1000, rotary=128,
              name="append_one"),
        # Prompts of odd lengths in single precision, adjacent pairs, half of each head rotated.
        _case("append", "float32", "int8", 4, 16, 4, 64, 32, new=513, old=100, rotary=32,
              interleaved=True, name="append_prompts_f32"),
        # Long prompts of a batch at once.
        _case("append", "bfloat16", "e4m3", 8, 32, 8, 128, 64, new=8191, rotary=128,
              name="append_prompts_8191"),
        # A short conversation's keys leave the cache.
        _case("read", "bfloat16", "e4m3", 1, 32, 8, 128, 16, new=1000, name="read_one_1000"),
        # Long sequences of a batch are moved out, but for the prompt that they began with.
        _case("read", "float16", "int8", 16, 32, 8, 128, 32, new=8191, old=500,
              name="read_batch_8191"),
        # One user's next token in a short conversation.
        _case("decode", "bfloat16", "e4m3", 1, 32, 8, 128, 16, old=1000, name="decode_one_1000"),
        # A decode step of a server: sequences of unlike lengths.
        _case("decode", "float16", "int8", 64, 32, 8, 128, 16, old=8191, name="decode_batch_64"),
        # A few users with long documents.
        _case("decode", "bfloat16", "e4m3", 4, 32, 8, 128, 64, old=131072, even=True,
              name="decode_long_131072"),
        # Drafted tokens of a batch are checked against caches of unlike lengths.
        _case("forward", "float16", "e4m3", 16, 32, 8, 128, 32, new=5, old=8191, even=True,
              name="forward_drafts_5"),
        # Prompts and next turns of unlike lengths in one step of a smaller model.
        _case("forward", "bfloat16", "int8", 7, 32, 4, 64, 16, new=2001, old=1000,
              name="forward_mixed_2001"),
        # Prompts in single precision.
        _case("forward", "float32", "int8", 2, 8, 8, 64, 16, new=1024, name="forward_f32_1024"),
        # One long prompt: the most products.
        _case("forward", "bfloat16", "e4m3", 1, 32, 8, 128, 64, new=16384,
              name="forward_prompt_16384"),
    ]


_GROUPED = [(32, 8), (16, 4), (16, 16), (32, 32), (8, 1), (32, 4), (12, 2), (8, 8), (40, 8),
            (32, 1)]


def _whole(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng):
    while True:
        op = rng.choice(["append", "read", "decode", "decode", "forward", "forward"])
        dtype = rng.choice(["float16", "bfloat16", "bfloat16", "float16", "float32"])
        code = rng.choice(["int8", "e4m3"])
        H, Hkv = rng.choice(_GROUPED)
        D = rng.choice([32, 64, 128, 128])
        page = rng.choice([16, 16, 32, 64, 128, 24])
        B = _whole(rng, 1, 32 if op == "forward" else 128)
        even = rng.random() < 0.3
        if op == "append":
            c = _case(op, dtype, code, B, H, Hkv, D, page,
                      new=1 if rng.random() < 0.4 else _whole(rng, 1, 8191),
                      old=_whole(rng, 1, 8191), even=even, rotary=rng.choice([D, D, D // 2, 0]),
                      interleaved=rng.random() < 0.3)
        elif op == "read":
            c = _case(op, dtype, code, B, H, Hkv, D, page, new=_whole(rng, 1, 8191),
                      old=_whole(rng, 1, 2048) - 1, even=even)
        elif op == "decode":
            c = _case(op, dtype, code, B, H, Hkv, D, page, old=_whole(rng, 1, 131072) - 1,
                      even=even)
        else:
            c = _case(op, dtype, code, B, H, Hkv, D, page, new=_whole(rng, 1, 16384),
                      old=_whole(rng, 1, 16384) - 1, even=even, causal=rng.random() < 0.85)
        w = work(c)
        keys = (c["new"] + c["old"]) * B * Hkv * D  # of the longest, for all of them
        scores = B * H * c["new"] * (c["new"] + c["old"]) if op == "forward" else 0
        if w["bytes"] < 1e9 and w["flops"] < (1.2e11 if dtype == "float32" else 2.2e12) \
                and keys < 6e8 and scores < 8.6e9:
            return c


def _lengths(c):
    """[(new tokens, keys before them)] of the sequences, in the order of their sizes."""
    B = c["B"]
    return [(c["new"] if c["even"] else max(1, c["new"] * (i + 1) // B),
             c["old"] if c["even"] else c["old"] * (B - i) // B) for i in range(B)]


def _filled(s, c, gen):
    """Codes and exponents of rows of a standard normal distribution, each by its largest element."""
    B, Hkv, D, page = c["B"], c["Hkv"], c["D"], c["page"]
    dev = torch.device("cuda")
    pages = s["pages"]
    codes = torch.empty((pages, page, Hkv, D), device=dev, dtype=torch.int8)
    exps = torch.empty((pages, Hkv, page), device=dev, dtype=torch.uint8)
    step = max(1, (1 << 26) // (page * Hkv * D))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        x = torch.randn((n, page, Hkv, D), device=dev, generator=gen)
        code, e = _quantised(c, x)
        codes[p:p + n] = code.view(torch.int8)
        exps[p:p + n] = e.transpose(1, 2)
    return codes.view(_code_type(c)), exps


def _code_type(c):
    return torch.int8 if c["code"] == "int8" else torch.float8_e4m3fn


def prepare(c, seed):
    dev = torch.device("cuda")
    dtype = getattr(torch, c["dtype"])
    gen = torch.Generator(device=dev).manual_seed(seed)

    def values(*shape):
        x = torch.empty(shape, device=dev, dtype=dtype)
        for part in x.split(max(1, (1 << 26) * shape[0] // max(1, x.numel()))):
            part.copy_(torch.randn(part.shape, device=dev, generator=gen))
        return x

    B, H, Hkv, D, page = (c[k] for k in ("B", "H", "Hkv", "D", "page"))
    lengths = _lengths(c)
    random.Random(seed).shuffle(lengths)
    new, total = [n for n, _ in lengths], [n + o for n, o in lengths]
    starts = [sum(new[:b]) for b in range(B + 1)]
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    s = {"case": c, "new": new, "total": total, "tokens": starts[B], "seq_lens": ints(total),
         "starts": ints(starts), "most_new": max(new), "most_keys": max(total)}

    # Pages in a random order, every sequence its own.
    own_pages = [-(-t // page) for t in total]
    s["pages"] = sum(own_pages)
    order = torch.randperm(s["pages"], device=dev, generator=gen).to(torch.int32)
    table = torch.zeros((B, max(own_pages)), dtype=torch.int32, device=dev)
    for b in range(B):
        at = sum(own_pages[:b])
        table[b, :own_pages[b]] = order[at:at + own_pages[b]]
    s["block_table"] = table
    s["k_cache"], s["k_exp"] = _filled(s, c, gen)
    s["v_cache"], s["v_exp"] = _filled(s, c, gen)

    if c["op"] == "append":
        # The projection's output: queries, keys and values of a token side by side.
        s["qkv"] = values(starts[B], H + 2 * Hkv, D)
        if c["rotary"]:
            half = c["rotary"] // 2
            rate = 1e4 ** (-torch.arange(half, device=dev, dtype=torch.float64) / half)
            angle = torch.arange(max(total), device=dev, dtype=torch.float64).unsqueeze(1) * rate
            s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        else:
            s["cos"] = s["sin"] = None
    elif c["op"] == "forward":
        s["q"] = values(starts[B], H, D)
    elif c["op"] == "decode":
        s["q"] = values(B, H, 1, D)
    return s


# ---- The operators in elementary operations ----

def _quantised(c, x):
    """Codes and exponent bytes of x [..., D], float32. The least exponent whose largest code is no
    smaller than the row's largest element comes from the bits of the two numbers."""
    bits = x.abs().amax(-1).view(torch.int32)
    top = torch.tensor(_TOP[c["code"]], device=x.device).view(torch.int32)
    e = (bits - top + ((1 << 23) - 1)) >> 23
    e = e.clamp(_LEAST, _MOST[c["code"], c["dtype"]])
    # 2^-e from its bits.
    y = x * ((127 - e) << 23).view(torch.float32).unsqueeze(-1)
    y = y.clamp(-_TOP[c["code"]], _TOP[c["code"]])
    code = y.round().to(torch.int8) if c["code"] == "int8" else y.to(torch.float8_e4m3fn)
    return code, (e + 127).to(torch.uint8)


def _rotated(c, x, cos, sin):
    """x [T, heads, D] with the first `rotary` elements of each head rotated; cos, sin [T, .]."""
    R = c["rotary"]
    if R == 0:
        return x
    first, second = (x[..., 0:R:2], x[..., 1:R:2]) if c["interleaved"] else \
        (x[..., :R // 2], x[..., R // 2:R])
    cos, sin = cos.unsqueeze(1), sin.unsqueeze(1)
    a, b = first * cos - second * sin, second * cos + first * sin
    turned = torch.stack((a, b), -1).flatten(-2) if c["interleaved"] else torch.cat((a, b), -1)
    return torch.cat((turned, x[..., R:]), -1)


def _split(s):
    H, Hkv = s["case"]["H"], s["case"]["Hkv"]
    return s["qkv"][:, :H], s["qkv"][:, H:H + Hkv], s["qkv"][:, H + Hkv:]


def _places(s):
    """Position, page and row in it of every token, on the GPU from the call's data."""
    starts, lens = s["starts"].long(), s["seq_lens"].long()
    t = torch.arange(s["tokens"], device=lens.device)
    b = torch.searchsorted(starts, t, right=True) - 1
    pos = lens[b] - starts[b + 1] + t
    page = s["block_table"][b, pos // s["case"]["page"]].long()
    return pos, page, pos % s["case"]["page"]


def _plain_append(s):
    c = s["case"]
    q, k, v = _split(s)
    pos, page, row = _places(s)
    cos, sin = (s["cos"][pos], s["sin"][pos]) if c["rotary"] else (None, None)
    k_code, k_e = _quantised(c, _rotated(c, k.float(), cos, sin))
    v_code, v_e = _quantised(c, v.float())
    s["k_cache"].view(torch.int8)[page, row] = k_code.view(torch.int8)
    s["v_cache"].view(torch.int8)[page, row] = v_code.view(torch.int8)
    s["k_exp"].transpose(1, 2)[page, row] = k_e
    s["v_exp"].transpose(1, 2)[page, row] = v_e
    return (_rotated(c, q.float(), cos, sin).to(q.dtype), s["k_cache"], s["v_cache"], s["k_exp"],
            s["v_exp"])


def _values(s, which, page, row):
    """The numbers in rows `row` of pages `page`, [..., Hkv, D] float32."""
    code = s[which + "_cache"].view(torch.int8)[page, row].view(_code_type(s["case"]))
    e = s[which + "_exp"].transpose(1, 2)[page, row].int()
    return code.float() * (e << 23).view(torch.float32).unsqueeze(-1)  # 2^(e - 127)


def _plain_read(s):
    dtype = getattr(torch, s["case"]["dtype"])
    _, page, row = _places(s)
    return _values(s, "k", page, row).to(dtype), _values(s, "v", page, row).to(dtype)


def _plain_attention(s):
    """All sequences at once, padded to the most tokens and the most keys."""
    c = s["case"]
    B, H, Hkv, D, page = (c[k] for k in ("B", "H", "Hkv", "D", "page"))
    G, n, L = H // Hkv, s["most_new"], s["most_keys"]
    lens, starts = s["seq_lens"].long(), s["starts"].long()
    q = s["q"].view(-1, H, D)
    at = torch.arange(L, device=q.device)
    used = s["block_table"][:, at // page].long()
    keys, vals = (_values(s, x, used, at % page) for x in "kv")
    i = torch.arange(n, device=q.device)
    token = (starts[:-1].unsqueeze(1) + i).clamp(max=q.shape[0] - 1)  # [B, n]
    here = i < (starts[1:] - starts[:-1]).unsqueeze(1)
    x = q[token].float().view(B, n, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B * Hkv, G * n, D)
    keys = keys.permute(0, 2, 3, 1).reshape(B * Hkv, D, L).contiguous()
    p = torch.bmm(x, keys).view(B, Hkv, G, n, L)
    p *= D ** -0.5
    last = lens.unsqueeze(1) - 1  # the last key that a token sees
    if c["causal"]:
        last = last - (starts[1:].unsqueeze(1) - 1 - starts[:-1].unsqueeze(1) - i).clamp(min=0)
    p.masked_fill_((at > last.unsqueeze(-1)).view(B, 1, 1, -1, L), -math.inf)
    m = p.amax(-1, keepdim=True)
    p -= m
    p.exp_()
    l = p.sum(-1, keepdim=True)
    vals = vals.permute(0, 2, 1, 3).reshape(B * Hkv, L, D).contiguous()
    o = torch.bmm(p.view(B * Hkv, G * n, L), vals).view(B, Hkv, G, n, D) / l
    lse = (m + torch.log(l)).squeeze(-1)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, n, H, D).to(q.dtype)[here]
    lse = lse.permute(0, 3, 1, 2).reshape(B, n, H)[here]
    return (o.view(s["q"].shape), lse.view(s["q"].shape[:-1]))


def _library():
    package = os.path.join(os.getcwd(), "cuflash-attn_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import cuflash_attn

    return cuflash_attn


def run(s):
    c = s["case"]
    if not own:
        return {"append": _plain_append, "read": _plain_read, "decode": _plain_attention,
                "forward": _plain_attention}[c["op"]](s)
    lib = _library()
    cache = (s["k_cache"], s["v_cache"], s["k_exp"], s["v_exp"])
    places = (s["block_table"], s["seq_lens"])
    if c["op"] == "append":
        q, k, v = _split(s)
        turned = lib.flash_attention_append_paged_q8(
            k, v, *cache, *places, s["starts"], q=q, cos=s["cos"], sin=s["sin"],
            interleaved=c["interleaved"])
        return (turned,) + cache
    if c["op"] == "read":
        return lib.flash_attention_read_paged_q8(*cache, *places, s["starts"], s["tokens"],
                                                 dtype=getattr(torch, c["dtype"]))
    if c["op"] == "decode":
        return lib.flash_attention_decode_paged_q8(s["q"], *cache, *places)
    return lib.flash_attention_forward_paged_q8(s["q"], *cache, *places, s["starts"],
                                                causal=c["causal"])


def work(c):
    H, Hkv, D = c["H"], c["Hkv"], c["D"]
    size = 4 if c["dtype"] == "float32" else 2
    lengths = _lengths(c)
    tokens = sum(n for n, _ in lengths)
    row = 2 * Hkv * (D + 1)  # a key's and a value's codes and exponents
    if c["op"] == "append":
        return {"bytes": tokens * ((2 * H + 2 * Hkv) * D * size + row + c["rotary"] * 4),
                "flops": tokens * ((H + Hkv) * c["rotary"] * 3 + 2 * Hkv * D * 3)}
    if c["op"] == "read":
        return {"bytes": tokens * (row + 2 * Hkv * D * size), "flops": tokens * 2 * Hkv * D}
    # Query and key pairs that the mask keeps, 4 D operations each; keys and values read once.
    keys = sum(n + o for n, o in lengths)
    causal = c["op"] == "forward" and c["causal"]
    pairs = sum(n * (n + o) - (n * (n - 1) // 2 if causal else 0) for n, o in lengths)
    return {"bytes": keys * row + tokens * H * (2 * D * size + 4), "flops": 4 * H * D * pairs}


# ---- The same from the definitions, in 64 bits ----

def _exact_codes(c, x):
    """Codes, as the numbers that they are, of rows x [..., D] in 64 bits."""
    top = _TOP[c["code"]]
    amax = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(amax / top))
    # Where the logarithm is rounded past a whole number.
    e = torch.where(amax > top * 2.0 ** e, e + 1, torch.where(amax <= top * 2.0 ** (e - 1), e - 1,
                                                              e))
    e = e.clamp(_LEAST, _MOST[c["code"], c["dtype"]])
    y = (x * 2.0 ** -e).clamp(-top, top)
    if c["code"] == "int8":
        return torch.round(y)
    # Three bits behind the leading one, steps of 2^-9 below 2^-6.
    _, exponent = torch.frexp(y)
    unit = 2.0 ** (exponent.double() - 1).clamp(min=-6) / 8
    return torch.round(y / unit) * unit


def exact(c, seed):
    s = prepare(c, seed)
    H, Hkv, D, page = (c[k] for k in ("H", "Hkv", "D", "page"))
    group = H // Hkv
    dev = s["k_cache"].device
    starts = s["starts"].tolist()

    def row(which, b, lo, hi):
        """Keys or values lo .. hi - 1 of sequence b, [hi - lo, Hkv, D] in 64 bits."""
        pages = s["block_table"][b, :-(-hi // page)].long()
        code = s[which + "_cache"].view(torch.int8)[pages].view(_code_type(c)).double()
        e = s[which + "_exp"][pages].double().permute(0, 2, 1).reshape(-1, Hkv, 1)
        return (code.reshape(-1, Hkv, D) * 2.0 ** (e - 127))[lo:hi]

    if c["op"] == "read":
        return tuple(torch.cat([row(w, b, t - n, t)
                                for b, (n, t) in enumerate(zip(s["new"], s["total"]))])
                     for w in "kv")
    if c["op"] == "append":
        rows = s["qkv"].double()
        if c["rotary"]:
            # Pair i of a head as a complex number, turned by cos + i sin of its position.
            pos = torch.cat([torch.arange(t - n, t, device=dev)
                             for n, t in zip(s["new"], s["total"])])
            turn = torch.complex(s["cos"].double(), s["sin"].double())[pos].unsqueeze(1)
            R = c["rotary"]
            re = torch.arange(R // 2, device=dev) * (2 if c["interleaved"] else 1)
            im = re + (1 if c["interleaved"] else R // 2)
            turned = torch.complex(rows[:, :H + Hkv, re], rows[:, :H + Hkv, im]) * turn
            rows[:, :H + Hkv, re], rows[:, :H + Hkv, im] = turned.real, turned.imag
        if c["code"] == "int8":  # whole numbers
            return rows[:, :H].contiguous(), None, None, None, None
        caches = [s["k_cache"].double(), s["v_cache"].double()]
        for b, (n, t) in enumerate(zip(s["new"], s["total"])):
            at = torch.arange(t - n, t, device=dev)
            to = s["block_table"][b, at // page].long()
            x = rows[starts[b]:starts[b + 1]]
            caches[0][to, at % page] = _exact_codes(c, x[:, H:H + Hkv])
            caches[1][to, at % page] = _exact_codes(c, x[:, H + Hkv:])
        return rows[:, :H].contiguous(), caches[0], caches[1], None, None
    q = s["q"].reshape(-1, H, D)
    out = torch.empty(q.shape, device=dev, dtype=torch.float64)
    lse = torch.empty(q.shape[:2], device=dev, dtype=torch.float64)
    for b, (n, total) in enumerate(zip(s["new"], s["total"])):
        keys, vals = row("k", b, 0, total), row("v", b, 0, total)
        t0 = starts[b]
        for h in range(Hkv):
            k, v = keys[:, h].contiguous(), vals[:, h].contiguous()
            for g in range(h * group, (h + 1) * group):
                for i in range(0, n, 8192):
                    part = slice(t0 + i, t0 + min(n, i + 8192))
                    p = torch.mm(q[part, g].double(), k.t())
                    p *= D ** -0.5
                    if c["op"] == "forward" and c["causal"]:
                        last = torch.arange(total - n + i, total - n + min(n, i + 8192),
                                            device=dev).unsqueeze(1)
                        p.masked_fill_(torch.arange(total, device=dev) > last, -math.inf)
                    z = torch.logsumexp(p, dim=1)
                    p -= z.unsqueeze(1)
                    p.exp_()
                    out[part, g], lse[part, g] = torch.mm(p, v), z
    return out.view(s["q"].shape), lse.view(s["q"].shape[:-1])
