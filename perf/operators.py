"""The paged-cache serving calls that the speed of this library is measured on.

Three operators that a server runs one after the other on one paged key/value cache: new tokens are
written into it with their rotation, several new tokens attend to it, and a batch whose sequences
share a prompt decodes from it. A case is one call. Fields:

  op      "append"   flash_attention_append_paged: rotates the new tokens' queries and keys and
                     writes keys and values to their pages
          "forward"  flash_attention_forward_paged: the new tokens' attention over the cache
          "shared"   flash_attention_decode_shared: one query per sequence, whose first `prefix`
                     keys are the same pages for the whole batch
  dtype   "float16", "bfloat16" or "float32"
  B, H, Hkv, D, page   sequences, query heads, key/value heads, head_dim, keys per page
  new     most new tokens of a sequence ("append", "forward"); sequence i of a batch has
          new (i + 1) / B of them, at least one, or all have `new` where `even`
  old     most keys that a sequence had before ("append", "forward"; old (B - i) / B of them), or
          that it has for itself beside the prefix ("shared"; old (i + 1) / B, at least one)
  causal  a token sees the keys up to its own ("forward")
  prefix  keys that the batch shares ("shared")
  rotary, interleaved   rotated elements of a head, and whether a pair is (2i, 2i + 1) or
          (i, i + rotary / 2) ("append")
"""

import math
import os
import random
import sys

import torch

own = False


def _case(op, dtype, B, H, Hkv, D, page, new=0, old=0, even=False, causal=True, prefix=0,
          rotary=0, interleaved=False, **name):
    return dict(name, op=op, dtype=dtype, B=B, H=H, Hkv=Hkv, D=D, page=page, new=new, old=old,
                even=even, causal=causal, prefix=prefix, rotary=rotary, interleaved=interleaved)


def listed():
    return [
        # One user's next token goes into the cache: the smallest call of a decode step.
        _case("append", "bfloat16", 1, 32, 8, 128, 16, new=1, old=1000, rotary=128,
              name="append_one"),
        # The next token of a batch, sequences of unlike lengths.
        _case("append", "float16", 64, 32, 8, 128, 16, new=1, old=8191, rotary=128,
              name="append_batch_64"),
        # Prompts of odd lengths in single precision, adjacent pairs, half of each head rotated.
        _case("append", "float32", 4, 16, 4, 64, 32, new=513, old=100, rotary=32,
              interleaved=True, name="append_prompts_f32"),
        # Long prompts of a batch at once: the most bytes.
        _case("append", "bfloat16", 8, 32, 8, 128, 64, new=8191, old=0, rotary=128,
              name="append_prompts_8191"),
        # The next turn of a chat: a few dozen tokens against a long cache.
        _case("forward", "bfloat16", 1, 32, 8, 128, 16, new=61, old=8192,
              name="forward_turn_61"),
        # Drafted tokens of a batch are checked against caches of unlike lengths.
        _case("forward", "float16", 16, 32, 8, 128, 32, new=5, old=8191, even=True,
              name="forward_drafts_5"),
        # Prompts and next turns of unlike lengths in one step of a smaller model.
        _case("forward", "bfloat16", 7, 32, 4, 64, 16, new=2001, old=1000,
              name="forward_mixed_2001"),
        # Prompts in single precision.
        _case("forward", "float32", 2, 8, 8, 64, 16, new=1024, old=0, name="forward_f32_1024"),
        # One long prompt: the most products.
        _case("forward", "bfloat16", 1, 32, 8, 128, 64, new=16384, old=0,
              name="forward_prompt_16384"),
        # A few answers to one prompt.
        _case("shared", "bfloat16", 4, 32, 8, 128, 16, prefix=1000, old=200,
              name="shared_four_1000"),
        # A batch behind one system prompt.
        _case("shared", "float16", 64, 32, 8, 128, 16, prefix=2048, old=1024,
              name="shared_batch_2048"),
        # Many questions to one long document.
        _case("shared", "bfloat16", 128, 32, 8, 128, 64, prefix=32768, old=512,
              name="shared_document_32768"),
    ]


_GROUPED = [(32, 8), (16, 4), (16, 16), (32, 32), (8, 1), (32, 4), (12, 2), (8, 8), (40, 8)]


def _whole(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng):
    while True:
        op = rng.choice(["append", "forward", "shared"])
        dtype = rng.choice(["float16", "bfloat16", "bfloat16", "float16", "float32"])
        H, Hkv = rng.choice(_GROUPED)
        D = rng.choice([32, 64, 128, 128])
        page = rng.choice([16, 16, 32, 64, 128, 24])
        if op == "append":
            rotary = rng.choice([D, D, D // 2, 0])
            c = _case(op, dtype, _whole(rng, 1, 128), H, Hkv, D, page,
                      new=1 if rng.random() < 0.4 else _whole(rng, 1, 8191),
                      old=_whole(rng, 1, 8191), even=rng.random() < 0.3, rotary=rotary,
                      interleaved=rng.random() < 0.3)
        elif op == "forward":
            new = _whole(rng, 1, 16384)
            c = _case(op, dtype, _whole(rng, 1, 32), H, Hkv, D, page, new=new,
                      old=_whole(rng, 1, 16384) - 1, even=rng.random() < 0.3,
                      causal=rng.random() < 0.85)
        else:
            c = _case(op, dtype, _whole(rng, 2, 128), H, Hkv, D, page,
                      prefix=_whole(rng, 128, 32768), old=_whole(rng, 1, 2048))
        w = work(c)
        # Single precision runs at a sixteenth of the 16-bit matrix rate.
        if w["bytes"] < 9e8 and w["flops"] < (1.2e11 if dtype == "float32" else 2.2e12):
            return c


def _lengths(c):
    """[(new tokens, keys before them)] of the sequences, in the order of their sizes."""
    B = c["B"]
    if c["op"] == "shared":
        return [(1, c["prefix"] + max(1, c["old"] * (i + 1) // B) - 1) for i in range(B)]
    return [(c["new"] if c["even"] else max(1, c["new"] * (i + 1) // B), c["old"] * (B - i) // B)
            for i in range(B)]


def prepare(c, seed):
    dev = torch.device("cuda")
    dtype = getattr(torch, c["dtype"])
    gen = torch.Generator(device=dev).manual_seed(seed)

    def values(*shape):
        x = torch.empty(shape, device=dev, dtype=dtype)
        for part in x.split(max(1, (1 << 26) * shape[0] // max(1, x.numel()))):
            part.copy_(torch.randn(part.shape, device=dev, generator=gen))
        return x

    B, H, Hkv, D, page, prefix = (c[k] for k in ("B", "H", "Hkv", "D", "page", "prefix"))
    lengths = _lengths(c)
    random.Random(seed).shuffle(lengths)
    new, total = [n for n, _ in lengths], [n + o for n, o in lengths]
    starts = [sum(new[:b]) for b in range(B + 1)]
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    s = {"case": c, "new": new, "total": total, "starts": starts, "seq_lens": ints(total),
         "query_starts": ints(starts)}

    # Pages in a random order. A sequence has its own page of every key behind the shared ones; a
    # shared prefix that ends inside a page leaves that page's first rows unused.
    first = prefix // page
    own_pages = [-(-t // page) - first for t in total]
    prefix_pages = -(-prefix // page)
    order = torch.randperm(sum(own_pages) + prefix_pages, device=dev, generator=gen)
    order = order.to(torch.int32)
    pages = order.numel()
    table = torch.zeros((B, max(own_pages) + first), dtype=torch.int32, device=dev)
    at = prefix_pages
    for b in range(B):
        table[b, first:first + own_pages[b]] = order[at:at + own_pages[b]]
        at += own_pages[b]
    s["block_table"], s["prefix_table"] = table, order[:prefix_pages].clone()
    s["k_cache"], s["v_cache"] = (values(pages, page, Hkv, D) for _ in range(2))

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
    else:
        s["q"] = values(B, H, 1, D)
    return s


def _split(s):
    H, Hkv = s["case"]["H"], s["case"]["Hkv"]
    return s["qkv"][:, :H], s["qkv"][:, H:H + Hkv], s["qkv"][:, H + Hkv:]


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


def _places(s):
    """Sequence, position, page and row in it of every token, on the GPU from the call's data."""
    starts, lens = s["query_starts"].long(), s["seq_lens"].long()
    t = torch.arange(s["starts"][-1], device=lens.device)
    b = torch.searchsorted(starts, t, right=True) - 1
    pos = lens[b] - starts[b + 1] + t
    page = s["block_table"][b, pos // s["case"]["page"]].long()
    return b, pos, page, pos % s["case"]["page"]


def _plain_append(s):
    c = s["case"]
    dtype = s["qkv"].dtype
    q, k, v = _split(s)
    _, pos, page, row = _places(s)
    cos, sin = (s["cos"][pos], s["sin"][pos]) if c["rotary"] else (None, None)
    s["k_cache"][page, row] = _rotated(c, k.float(), cos, sin).to(dtype)
    s["v_cache"][page, row] = v
    return _rotated(c, q.float(), cos, sin).to(dtype), s["k_cache"], s["v_cache"]


def _plain_forward(s):
    c = s["case"]
    H, Hkv, D, page = (c[k] for k in ("H", "Hkv", "D", "page"))
    q = s["q"]
    T, G = q.shape[0], H // Hkv
    out = torch.empty_like(q)
    lse = torch.empty((T, H), device=q.device, dtype=torch.float32)
    for b in range(c["B"]):
        n, total, t0 = s["new"][b], s["total"][b], s["starts"][b]
        used = s["block_table"][b, :-(-total // page)].long()
        keys, vals = (s[x][used].reshape(-1, Hkv, D)[:total].float()
                      for x in ("k_cache", "v_cache"))
        hidden = None
        if c["causal"]:
            pos = torch.arange(total - n, total, device=q.device)
            hidden = torch.arange(total, device=q.device) > pos.unsqueeze(1)
        for h in range(Hkv):
            x = q[t0:t0 + n, h * G:(h + 1) * G].float().transpose(0, 1).reshape(G * n, D)
            p = (torch.mm(x, keys[:, h].t().contiguous()) * D ** -0.5).view(G, n, total)
            if hidden is not None:
                p.masked_fill_(hidden, -math.inf)
            m = p.amax(-1, keepdim=True)
            p = torch.exp(p - m)
            l = p.sum(-1, keepdim=True)
            o = torch.mm(p.view(G * n, total), vals[:, h].contiguous()).view(G, n, D) / l
            out[t0:t0 + n, h * G:(h + 1) * G] = o.transpose(0, 1).to(q.dtype)
            lse[t0:t0 + n, h * G:(h + 1) * G] = (m + torch.log(l)).squeeze(-1).t()
    return out, lse


def _plain_shared(s):
    c = s["case"]
    B, H, Hkv, D, page, prefix = (c[k] for k in ("B", "H", "Hkv", "D", "page", "prefix"))
    q, G = s["q"], H // Hkv
    x = q.view(B, Hkv, G, D).float() * D ** -0.5
    # The shared keys once for the batch, the rest padded to the longest.
    shared = [s[n][s["prefix_table"].long()].reshape(-1, Hkv, D)[:prefix].float()
              for n in ("k_cache", "v_cache")]
    at = torch.arange(prefix, max(s["total"]), device=q.device)
    used = s["block_table"][:, at // page].long()
    rest = [s[n][used, at % page].float() for n in ("k_cache", "v_cache")]
    hidden = at >= s["seq_lens"].unsqueeze(1)
    out = torch.empty((B, Hkv, G, D), device=q.device, dtype=q.dtype)
    lse = torch.empty((B, Hkv, G), device=q.device, dtype=torch.float32)
    for h in range(Hkv):
        xh = x[:, h].contiguous()
        p = torch.mm(xh.view(B * G, D), shared[0][:, h].t().contiguous()).view(B, G, prefix)
        r = torch.bmm(xh, rest[0][:, :, h].transpose(1, 2).contiguous())
        r.masked_fill_(hidden.unsqueeze(1), -math.inf)
        p = torch.cat((p, r), -1)
        m = p.amax(-1, keepdim=True)
        p = torch.exp(p - m)
        l = p.sum(-1, keepdim=True)
        o = torch.mm(p[..., :prefix].reshape(B * G, prefix), shared[1][:, h].contiguous())
        o = o.view(B, G, D) + torch.bmm(p[..., prefix:].contiguous(),
                                        rest[1][:, :, h].contiguous())
        out[:, h] = (o / l).to(q.dtype)
        lse[:, h] = (m + torch.log(l)).squeeze(-1)
    return out.view(B, H, 1, D), lse.view(B, H, 1)


def _library():
    package = os.path.join(os.getcwd(), "cuflash-attn_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import cuflash_attn

    return cuflash_attn


def run(s):
    c = s["case"]
    if not own:
        return {"append": _plain_append, "forward": _plain_forward,
                "shared": _plain_shared}[c["op"]](s)
    lib = _library()
    cache = (s["k_cache"], s["v_cache"])
    if c["op"] == "append":
        q, k, v = _split(s)
        turned = lib.flash_attention_append_paged(
            k, v, *cache, s["block_table"], s["seq_lens"], s["query_starts"], q=q, cos=s["cos"],
            sin=s["sin"], interleaved=c["interleaved"])
        return (turned,) + cache
    if c["op"] == "forward":
        return lib.flash_attention_forward_paged(s["q"], *cache, s["block_table"], s["seq_lens"],
                                                 s["query_starts"], causal=c["causal"])
    return lib.flash_attention_decode_shared(s["q"], *cache, s["prefix_table"], c["prefix"],
                                             s["block_table"], s["seq_lens"])


def work(c):
    H, Hkv, D = c["H"], c["Hkv"], c["D"]
    size = 4 if c["dtype"] == "float32" else 2
    lengths = _lengths(c)
    tokens = sum(n for n, _ in lengths)
    if c["op"] == "append":
        # Every new row is read and written once, and a token's angles are read.
        heads = H + (H + 4 * Hkv)
        return {"bytes": tokens * (heads * D * size + c["rotary"] * 4),
                "flops": tokens * (H + Hkv) * c["rotary"] * 3}
    # Query and key pairs that the mask keeps, 4 D operations each; keys and values read once.
    if c["op"] == "forward":
        pairs = sum(n * (n + o) - (n * (n - 1) // 2 if c["causal"] else 0) for n, o in lengths)
        keys = sum(n + o for n, o in lengths)
    else:
        pairs = sum(n + o for n, o in lengths)
        keys = c["prefix"] + pairs - c["B"] * c["prefix"]
    return {"bytes": 2 * keys * Hkv * D * size + tokens * H * (2 * D * size + 4),
            "flops": 4 * H * D * pairs}


def exact(c, seed):
    s = prepare(c, seed)
    H, Hkv, D, page, prefix = (c[k] for k in ("H", "Hkv", "D", "page", "prefix"))
    group = H // Hkv
    dev = s["k_cache"].device
    if c["op"] == "append":
        caches = [s["k_cache"].double(), s["v_cache"].double()]
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
        for b in range(c["B"]):
            for p in range((s["total"][b] - s["new"][b]) // page, -(-s["total"][b] // page)):
                lo = max(p * page, s["total"][b] - s["new"][b])
                hi = min((p + 1) * page, s["total"][b])
                t = s["starts"][b + 1] - s["total"][b]
                n = int(s["block_table"][b, p])
                caches[0][n, lo - p * page:hi - p * page] = rows[t + lo:t + hi, H:H + Hkv]
                caches[1][n, lo - p * page:hi - p * page] = rows[t + lo:t + hi, H + Hkv:]
        return (rows[:, :H].contiguous(),) + tuple(caches)
    q = s["q"].reshape(-1, H, D)
    out = torch.empty(q.shape, device=dev, dtype=torch.float64)
    lse = torch.empty(q.shape[:2], device=dev, dtype=torch.float64)
    for b in range(c["B"]):
        n, total, t0 = s["new"][b], s["total"][b], s["starts"][b]
        pages = s["block_table"][b, :-(-total // page)].long()
        keys, vals = (s[x][pages].reshape(-1, Hkv, D)[:total] for x in ("k_cache", "v_cache"))
        if prefix:
            at = s["prefix_table"].long()
            keys, vals = (torch.cat((s[x][at].reshape(-1, Hkv, D)[:prefix], y[prefix:]))
                          for x, y in (("k_cache", keys), ("v_cache", vals)))
        for h in range(Hkv):
            k, v = keys[:, h].double(), vals[:, h].double()
            for g in range(h * group, (h + 1) * group) if n > 1 else [slice(h * group,
                                                                            (h + 1) * group)]:
                x = q[t0:t0 + n, g].double().reshape(-1, D)
                p = torch.mm(x, k.t())
                p *= D ** -0.5
                if c["causal"] and n > 1:
                    last = torch.arange(total - n, total, device=dev).unsqueeze(1)
                    p.masked_fill_(torch.arange(total, device=dev) > last, -math.inf)
                z = torch.logsumexp(p, dim=1)
                p -= z.unsqueeze(1)
                p.exp_()
                o = torch.mm(p, v)
                if n > 1:
                    out[t0:t0 + n, g], lse[t0:t0 + n, g] = o, z
                else:
                    out[t0, g], lse[t0, g] = o, z
    if c["op"] == "shared":
        return out.unsqueeze(2), lse.unsqueeze(2)
    return out, lse
