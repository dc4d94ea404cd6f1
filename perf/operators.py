"""Timed cases of the operators around a paged key/value cache: rotary positions, writing new tokens into the cache,
attention of new tokens over it, and the bookkeeping of its pages.

A case is a dict of plain values; `op` names the operator:

  rotary     one layer's queries and keys are rotated by their positions (`train`: and the gradient comes back)
  append     one layer's new keys and values go to their pages (`rotary`: rotated on the way, the queries as well)
  attention  one layer's new tokens attend to everything their sequences hold, themselves included
  branch     sequences are dropped, replaced by forks of others, and given room for their next tokens
  compact    the pages in use move to the front of the pool

`run` with `own` false is the plain form: elementary torch operations in 32 bits (angles in 64), rounded once. With `own`
true it makes the calls of spargeattn_b200 that a program makes.

The cache: pages [num_pages, kv_heads, page_size, D] of keys and of values, page_table [sequences, width] int32 (-1: no
page), seq_lens [sequences] int32 (tokens held, the new ones included), ref_counts [num_pages] int32. New tokens are packed
[tokens, heads, D]; sequence i has rows cu_seqlens[i] to cu_seqlens[i + 1], its last tokens.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------------------- the cases
def _rotary(name, B, N, Hq, Hkv, D, rot, dtype="bf16", interleaved=False, axes=1, layout="NHD", far=0, factor=1.0, train=False):
    return dict(name=name, op="rotary", B=B, N=N, Hq=Hq, Hkv=Hkv, D=D, rot=rot, dtype=dtype, interleaved=interleaved, axes=axes,
                layout=layout, far=far, factor=factor, train=train)


def _append(name, B, chunk, length, Hq, Hkv, D, page, dtype="bf16", rotary=True, interleaved=False):
    return dict(name=name, op="append", B=B, chunk=chunk, length=length, Hq=Hq, Hkv=Hkv, D=D, page=page, dtype=dtype, rotary=rotary,
                interleaved=interleaved)


def _attention(name, B, chunk, length, Hq, Hkv, D, page, dtype="bf16", causal=True, lse=False):
    return dict(name=name, op="attention", B=B, chunk=chunk, length=length, Hq=Hq, Hkv=Hkv, D=D, page=page, dtype=dtype,
                causal=causal, lse=lse)


def _pool(name, op, layers, pages, page, Hkv, D, sequences, length, dtype="bf16"):
    return dict(name=name, op=op, layers=layers, pages=pages, page=page, Hkv=Hkv, D=D, sequences=sequences, length=length,
                dtype=dtype)


def listed():
    return [
        # one step of eight conversations far into a context four times the trained one: launch and latency count
        _rotary("rotary_step", 8, 1, 32, 8, 128, 128, far=100_003, factor=4.0),
        # a layer of a video transformer in training: frame, row and column positions, adjacent pairs, and the gradient
        _rotary("rotary_video_train", 1, 32760, 12, 12, 128, 128, interleaved=True, axes=3, layout="HND", train=True),
        # a ragged prompt of a model that rotates half of each head
        _rotary("rotary_partial_prompt", 1, 4097, 16, 4, 128, 64, dtype="fp16", far=511),
        # one token for each of 64 conversations, rotated and written in the same call
        _append("append_step", 64, 1, 4096, 32, 8, 128, 16),
        # chunks of prompts, already rotated
        _append("append_chunks", 7, 2047, 6000, 16, 16, 64, 64, dtype="fp16", rotary=False),
        # one short conversation: the smallest call
        _attention("decode_one", 1, 1, 777, 8, 2, 128, 16),
        # a serving batch, one token each, ragged lengths
        _attention("decode_batch", 64, 1, 8191, 32, 8, 128, 16),
        # two very long contexts, eight query heads to a key head: few rows, a long axis
        _attention("decode_long", 2, 1, 131_075, 16, 2, 128, 64, lse=True),
        # chunks of prompts of different lengths beside single tokens, small heads
        _attention("chunks_ragged", 9, 700, 5003, 16, 16, 64, 32, dtype="fp16"),
        # a long prompt's chunk over what came before it: the largest
        _attention("chunk_long", 1, 4096, 20_477, 32, 8, 128, 64, lse=True),
        # beams: a third of the sequences is replaced by forks of the others
        _pool("beams", "branch", 8, 2048, 32, 8, 128, 48, 900),
        # a fragmented pool is packed before it is shrunk
        _pool("pack", "compact", 8, 2048, 32, 8, 128, 64, 640),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "append", "attention", "attention", "branch", "compact"])
    D, dtype = rng.choice([64, 128]), rng.choice(["bf16", "fp16"])
    Hkv = rng.choice([1, 2, 4, 8])
    Hq = Hkv * rng.choice([1, 2, 4, 5, 8])
    page = rng.choice([16, 32, 64, 128])
    if op == "rotary":
        axes = rng.choice([1, 1, 3])
        N = _log(rng, 1, 20_000)
        c = _rotary("", 1 if N > 64 else rng.randint(1, 64), N, Hq, Hkv, D, D if axes == 3 else rng.choice([D, D // 2]),
                    rng.choice(["bf16", "fp16", "fp32"]), rng.random() < 0.5, axes, rng.choice(["NHD", "HND"]),
                    0 if axes == 3 else rng.randint(0, 200_000), rng.choice([1.0, 2.0, 8.0]), rng.random() < 0.4)
    elif op == "append":
        chunk = rng.choice([1, _log(rng, 2, 2000)])
        B = _log(rng, 1, 128) if chunk == 1 else rng.randint(1, 8)
        c = _append("", B, chunk, max(chunk, _log(rng, 8, 8000)), Hq, Hkv, D, page, dtype, rng.random() < 0.6, rng.random() < 0.5)
    elif op == "attention":
        chunk = rng.choice([1, 1, _log(rng, 2, 12), _log(rng, 12, 3000)])
        B = _log(rng, 1, 48) if chunk <= 12 else rng.randint(1, 6)
        length = max(chunk, _log(rng, 8, 60_000 if B <= 3 and chunk <= 12 else 6000))
        c = _attention("", B, chunk, length, Hq, Hkv, D, page, dtype, rng.random() < 0.85, rng.random() < 0.5)
    else:
        sequences = rng.randint(6, 48)
        length = _log(rng, 100, 900)
        need = sequences * (-(-length // page) + 2) * 3 // 2
        c = _pool("", op, rng.randint(1, 6), need + rng.randint(0, 200), page, min(Hkv, 4), D, sequences, length, dtype)
    del c["name"]
    return c


def _spread(n, top, least):
    """n whole numbers from top down towards least, ragged, the first one top."""
    return [max(least, int(round(least + (top - least) * (1.0 - 0.8 * ((0.618033988749895 * i) % 1.0))))) for i in range(n)]


def _chunks(case):
    return [1] * case["B"] if case["chunk"] == 1 else _spread(case["B"], case["chunk"], 1)


def _lengths(case):
    return [max(a, b) for a, b in zip(_spread(case["B"], case["length"], 1), _chunks(case))]


# --------------------------------------------------------------------------------------------------------- the inputs
def _cache(case, lengths, g, spare):
    """Pages in random order for these sequences, a table of them, and the lengths."""
    ps, dt = case["page"], DTYPES[case["dtype"]]
    used = [-(-n // ps) for n in lengths]
    pages, width = sum(used) + spare, max(used) + 1
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    first = [sum(used[:i]) for i in range(len(used))]
    at = torch.arange(width, device="cuda")
    idx = torch.tensor(first, device="cuda")[:, None] + at
    here = at < torch.tensor(used, device="cuda")[:, None]
    table = torch.where(here, order[idx.clamp(max=pages - 1)], torch.full_like(order[:1], -1))
    shape = (pages, case["Hkv"], ps, case["D"])
    return dict(k_pages=torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dt),
                v_pages=torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dt),
                page_table=table.contiguous(), seq_lens=torch.tensor(lengths, dtype=torch.int32, device="cuda"))


def _cumulated(chunks):
    return torch.tensor([sum(chunks[:i]) for i in range(len(chunks) + 1)], dtype=torch.int32, device="cuda")


def _frequencies(rot, factor):
    return 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot) / factor


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    op, dt = case["op"], DTYPES[case["dtype"]]
    rand = lambda *s: torch.randn(s, generator=g, device="cuda", dtype=torch.float32).to(dt)  # noqa: E731
    s = dict(case)
    if op == "rotary":
        B, N, D, rot = case["B"], case["N"], case["D"], case["rot"]
        shape = (lambda H: (B, H, N, D)) if case["layout"] == "HND" else (lambda H: (B, N, H, D))
        s |= dict(q=rand(*shape(case["Hq"])), k=rand(*shape(case["Hkv"])), frequencies=_frequencies(rot, case["factor"]))
        n = torch.arange(N, dtype=torch.int32, device="cuda")
        if case["axes"] == 3:   # a grid of frames, rows and columns
            w, h = 52, 30
            s |= dict(positions=torch.stack([n // (w * h), n // w % h, n % w]), sections=[rot // 2 - 2 * (rot // 6), rot // 6, rot // 6])
        else:
            s |= dict(positions=case["far"] + n + 17 * torch.arange(B, dtype=torch.int32, device="cuda")[:, None], sections=None)
        if case["train"]:
            s |= dict(gq=rand(*shape(case["Hq"])), gk=rand(*shape(case["Hkv"])))
            s["q"].requires_grad_(), s["k"].requires_grad_()
        return s
    if op in ("append", "attention"):
        chunks, lengths = _chunks(case), _lengths(case)
        T = sum(chunks)
        s |= _cache(case, lengths, g, 3)
        s |= dict(cu_seqlens=None if case["chunk"] == 1 else _cumulated(chunks), T=T, max_length=max(lengths), q=rand(T, case["Hq"], case["D"]))
        if op == "append":
            s |= dict(k=rand(T, case["Hkv"], case["D"]), v=rand(T, case["Hkv"], case["D"]),
                      frequencies=_frequencies(case["D"], 1.0) if case["rotary"] else None)
        return s
    # branch, compact: a pool that has been in use for a while
    P, n, ps = case["pages"], case["sequences"], case["page"]
    lengths = _spread(n, case["length"], 1)
    used = [-(-x // ps) for x in lengths]
    width = max(used) + 3
    order = torch.randperm(P, generator=g, device="cuda").to(torch.int32)
    idx = torch.tensor([sum(used[:i]) for i in range(n)], device="cuda")[:, None] + torch.arange(width, device="cuda")
    here = torch.arange(width, device="cuda") < torch.tensor(used, device="cuda")[:, None]
    table = torch.where(here, order[idx.clamp(max=P - 1)], torch.full_like(order[:1], -1)).contiguous()
    refs = torch.zeros(P, dtype=torch.int32, device="cuda")
    refs[order[: sum(used)].long()] = 1
    s |= dict(pages_=rand(case["layers"], 2, P, case["Hkv"], ps, case["D"]), page_table=table, ref_counts=refs,
              seq_lens=torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    if op == "branch":
        order = torch.randperm(n, generator=g, device="cuda").to(torch.int32)
        k = n // 3
        s |= dict(dst=order[:k].contiguous(), src=order[k + torch.randint(0, n - k, (k,), generator=g, device="cuda")].contiguous(),
                  new_tokens=torch.zeros(n, dtype=torch.int32, device="cuda"))
        s["new_tokens"][s["dst"].long()] = ps + 1
    else:
        s |= dict(table_before=table.clone(), refs_before=refs.clone())
    return s


# --------------------------------------------------------------------------------------------------- the plain forms
def _angles(positions, frequencies, sections):
    """Phases in 64 bits, reduced to one turn, then cosines and sines in 32: [..., rot / 2]."""
    if sections is None:
        a = positions.double()[..., None] * frequencies
    else:
        axis = torch.repeat_interleave(torch.arange(len(sections), device=positions.device),
                                       torch.tensor(sections, device=positions.device), output_size=frequencies.numel())
        a = positions.double()[axis].movedim(0, -1) * frequencies
    a = torch.remainder(a, 2.0 * math.pi).float()
    return a.cos(), a.sin()


def _turn(x, cos, sin, interleaved):
    """x [..., D] rotated in 32 bits; cos and sin broadcast against [..., rot / 2]."""
    half = cos.shape[-1]
    f = x.float()
    head, rest = f[..., : 2 * half], f[..., 2 * half:]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., :half], head[..., half:])
    u, w = a * cos - b * sin, a * sin + b * cos
    y = torch.stack([u, w], -1).flatten(-2) if interleaved else torch.cat([u, w], -1)
    return torch.cat([y, rest], -1).to(x.dtype)


def _rows(s):
    """For each packed token: its sequence and its position there."""
    T, dev = s["T"], s["seq_lens"].device
    if s["cu_seqlens"] is None:
        seq = torch.arange(T, device=dev)
        return seq, s["seq_lens"].long() - 1
    cu = s["cu_seqlens"].long()
    seq = torch.searchsorted(cu, torch.arange(T, device=dev), right=True) - 1
    return seq, s["seq_lens"].long()[seq] - cu[seq + 1] + torch.arange(T, device=dev)


def _plain_rotary(s):
    cos, sin = _angles(s["positions"], s["frequencies"], s["sections"])
    cos, sin = (t.unsqueeze(-3 if s["layout"] == "HND" else -2) for t in (cos, sin))
    out = dict(q=_turn(s["q"].detach(), cos, sin, s["interleaved"]), k=_turn(s["k"].detach(), cos, sin, s["interleaved"]))
    if s["train"]:   # the gradient turns back
        out |= dict(dq=_turn(s["gq"], cos, -sin, s["interleaved"]), dk=_turn(s["gk"], cos, -sin, s["interleaved"]))
    return out


def _plain_append(s):
    seq, pos = _rows(s)
    q, k = s["q"], s["k"]
    if s["rotary"]:
        cos, sin = (t[:, None] for t in _angles(pos, s["frequencies"], None))
        q, k = _turn(q, cos, sin, s["interleaved"]), _turn(k, cos, sin, s["interleaved"])
    page = s["page_table"][seq, pos // s["page"]].long()
    s["k_pages"][page, :, pos % s["page"]] = k
    s["v_pages"][page, :, pos % s["page"]] = s["v"]
    return dict(k_pages=s["k_pages"], v_pages=s["v_pages"], **({"q": q} if s["rotary"] else {}))


def _plain_attention(s):
    B, Hq, Hkv, D, ps, n = s["B"], s["Hq"], s["Hkv"], s["D"], s["page"], s["chunk"]
    dev, G = s["q"].device, Hq // Hkv
    np_ = -(-s["max_length"] // ps)
    pages = s["page_table"][:, :np_].clamp(min=0).long()
    k, v = (s[w][pages].transpose(1, 2).reshape(B, Hkv, np_ * ps, D).float() for w in ("k_pages", "v_pages"))
    lens = s["seq_lens"].long()
    cu = s["cu_seqlens"].long() if s["cu_seqlens"] is not None else torch.arange(B + 1, device=dev)
    count = cu[1:] - cu[:-1]
    i = torch.arange(n, device=dev)
    row = (cu[:-1, None] + i).clamp(max=s["T"] - 1)                                   # [B, n]
    q = s["q"][row].float().view(B, n, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * n, D)
    last = (lens - count)[:, None] + i if s["causal"] else (lens - 1)[:, None].expand(B, n)
    key = torch.arange(np_ * ps, device=dev)
    see = (key <= last[..., None]) & (key < lens[:, None, None]) & (i < count[:, None])[..., None]  # [B, n, K]
    x = torch.matmul(q, k.transpose(-1, -2)).mul_(D ** -0.5).view(B, Hkv, G, n, -1)
    x = x.masked_fill_(~see[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True).clamp_(min=-1e30)
    x = x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(B, Hkv, G * n, -1), v).view(B, Hkv, G, n, D) / total.clamp(min=1e-30)
    lse = (top + total.log()).squeeze(-1)
    here = (i < count[:, None])
    out = torch.zeros(s["T"], Hq, D, dtype=s["q"].dtype, device=dev)
    where = torch.where(here, row, s["T"])                                            # rows of no token go behind the last
    out = torch.cat([out, out[:1]])
    out[where] = o.permute(0, 3, 1, 2, 4).reshape(B, n, Hq, D).to(out.dtype)
    if not s["lse"]:
        return out[:-1]
    l2 = torch.zeros(s["T"] + 1, Hq, dtype=torch.float32, device=dev)
    l2[where] = lse.permute(0, 3, 1, 2).reshape(B, n, Hq)
    return out[:-1], l2[:-1]


def _plain_free(s, rows):
    rows = rows.long()
    held = s["page_table"][rows]
    held = held[held >= 0].long()
    s["ref_counts"].index_add_(0, held, torch.full_like(held, -1, dtype=torch.int32))
    s["page_table"][rows] = -1
    s["seq_lens"][rows] = 0


def _plain_branch(s):
    ps = s["page"]
    table, lens, refs, dst, src = s["page_table"], s["seq_lens"], s["ref_counts"], s["dst"].long(), s["src"].long()
    _plain_free(s, dst)
    # forks share the full pages; a page that is not full is copied to the lowest free one
    rows, n = table[src], lens[src].long()
    part = (n % ps != 0).nonzero().squeeze(1)
    free = (refs == 0).nonzero().squeeze(1)
    new, at = free[: part.numel()], n[part] // ps
    old = rows[part, at].long()
    rows[part, at] = new.int()
    s["pages_"][:, :, new] = s["pages_"][:, :, old]
    table[dst], lens[dst] = rows, n.int()
    held = rows[rows >= 0].long()
    refs.index_add_(0, held, torch.ones_like(held, dtype=torch.int32))
    # room for the forks' next tokens: the lowest free pages, in the order of the sequences
    grown, at = lens + s["new_tokens"], torch.arange(table.shape[1], device=table.device)
    lacks = (at >= ((lens + ps - 1) // ps)[:, None]) & (at < ((grown + ps - 1) // ps)[:, None])
    new = (refs == 0).nonzero().squeeze(1)[: lacks.sum()]
    table[lacks] = new.int()
    refs[new] = 1
    lens.copy_(grown)
    return s["pages_"], table, lens, refs


def _plain_compact(s):
    refs, table = s["ref_counts"], s["page_table"]
    live = refs > 0
    count = live.sum()
    at = torch.arange(refs.numel(), device=refs.device)
    src, dst = (live & (at >= count)).nonzero().squeeze(1), (~live & (at < count)).nonzero().squeeze(1)
    s["pages_"][:, :, dst] = s["pages_"][:, :, src]
    to = at.int()
    to[src] = dst.int()
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()], table))
    refs[dst] = refs[src]
    refs[src] = 0
    return s["pages_"], table, refs, count.int().view(1)


# -------------------------------------------------------------------------------------------------------------- a pass
def _back_to_before(s):
    """A program that gave up its latest step: the bookkeeping of a pool is what it was before the pass."""
    if s["op"] == "compact":
        s["page_table"].copy_(s["table_before"])
        s["ref_counts"].copy_(s["refs_before"])


def _own(s):
    import spargeattn_b200 as S
    op = s["op"]
    if op == "rotary":
        q, k = S.apply_rotary(s["q"], s["k"], s["positions"], s["frequencies"], interleaved=s["interleaved"], sections=s["sections"],
                              tensor_layout=s["layout"])
        out = dict(q=q, k=k)
        if s["train"]:
            dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["gq"], s["gk"]))
            out = dict(q=q.detach(), k=k.detach(), dq=dq, dk=dk)
        return out
    if op == "append":
        q = S.append_kv(s["k"], s["v"], s["k_pages"], s["v_pages"], s["page_table"], s["seq_lens"], s["cu_seqlens"],
                        q=s["q"] if s["rotary"] else None, frequencies=s["frequencies"], interleaved=s["interleaved"])
        return dict(k_pages=s["k_pages"], v_pages=s["v_pages"], **({"q": q} if s["rotary"] else {}))
    if op == "attention":
        return S.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["seq_lens"], s["cu_seqlens"],
                                 max_chunk=s["chunk"], is_causal=s["causal"], return_lse=s["lse"])
    if op == "branch":
        S.free_sequences(s["page_table"], s["seq_lens"], s["ref_counts"], s["dst"], s["page"])
        S.fork_sequences(s["pages_"], s["page_table"], s["seq_lens"], s["ref_counts"], s["src"], s["dst"])
        S.allocate_pages(s["page_table"], s["seq_lens"], s["ref_counts"], s["new_tokens"], s["page"])
        return s["pages_"], s["page_table"], s["seq_lens"], s["ref_counts"]
    count = S.compact_pages(s["pages_"], s["page_table"], s["ref_counts"])
    return s["pages_"], s["page_table"], s["ref_counts"], count


def run(state):
    _back_to_before(state)
    if own:
        return _own(state)
    return {"rotary": _plain_rotary, "append": _plain_append, "attention": _plain_attention, "branch": _plain_branch,
            "compact": _plain_compact}[state["op"]](state)


# ------------------------------------------------------------------------------------------------------------ the work
def work(case):
    op, e = case["op"], 4 if case["dtype"] == "fp32" else 2
    if op == "rotary":
        x = case["B"] * case["N"] * (case["Hq"] + case["Hkv"])
        passes = 2 if case["train"] else 1
        return {"bytes": passes * 2.0 * x * case["D"] * e + 4.0 * case["B"] * case["N"] * case["axes"], "flops": passes * 3.0 * x * case["rot"]}
    if op == "append":
        T, D = sum(_chunks(case)), case["D"]
        x = T * case["Hkv"] * D * 2 + (T * case["Hq"] * D if case["rotary"] else 0)
        return {"bytes": 2.0 * x * e + 8.0 * T, "flops": 3.0 * T * (case["Hq"] + case["Hkv"]) * D if case["rotary"] else 0.0}
    if op == "attention":
        ch, ln, D = _chunks(case), _lengths(case), case["D"]
        seen = sum(c * n - (c * (c - 1) // 2 if case["causal"] else 0) for c, n in zip(ch, ln))
        held = sum(ln) * case["Hkv"] * D * 2 * e
        return {"bytes": held + 2.0 * sum(ch) * case["Hq"] * D * e + (4.0 * sum(ch) * case["Hq"] if case["lse"] else 0.0),
                "flops": 4.0 * seen * case["Hq"] * D}
    page = case["layers"] * 2 * case["Hkv"] * case["page"] * case["D"] * e
    lengths, ps = _spread(case["sequences"], case["length"], 1), case["page"]
    used = sum(-(-n // ps) for n in lengths)
    if op == "branch":
        forks = case["sequences"] // 3
        return {"bytes": 2.0 * page * forks * sum(n % ps != 0 for n in lengths) / len(lengths) + 8.0 * (case["pages"] + used), "flops": 0.0}
    return {"bytes": 2.0 * page * used * (case["pages"] - used) / case["pages"] + 8.0 * (case["pages"] + used), "flops": 0.0}


# ------------------------------------------------------------------------------------------------- in 64 bits, by itself
def _exact_rotate(x, phase, interleaved):
    """x [..., D] by the complex product with exp(i phase), phase [..., rot / 2]."""
    r = 2 * phase.shape[-1]
    x = x.double()
    z = torch.complex(x[..., 0:r:2], x[..., 1:r:2]) if interleaved else torch.complex(x[..., : r // 2], x[..., r // 2: r])
    z = z * torch.polar(torch.ones_like(phase), phase)
    y = torch.view_as_real(z).flatten(-2) if interleaved else torch.cat([z.real, z.imag], -1)
    return torch.cat([y, x[..., r:]], -1)


def _exact_rotary(s):
    freq = s["frequencies"]
    if s["sections"] is None:
        pos = s["positions"].double()[..., None].expand(*s["positions"].shape, freq.numel())
    else:
        pos = torch.cat([s["positions"][a].double()[:, None].expand(-1, n) for a, n in enumerate(s["sections"])], -1)
    phase = (pos * freq).unsqueeze(-2)                                                # [..., N, 1, rot / 2]

    def one(x, sign):
        hnd = s["layout"] == "HND"
        t = x.detach().transpose(1, 2) if hnd else x.detach()
        y = _exact_rotate(t, sign * phase, s["interleaved"])
        return y.transpose(1, 2).contiguous() if hnd else y

    out = dict(q=one(s["q"], 1.0), k=one(s["k"], 1.0))
    if s["train"]:
        out |= dict(dq=one(s["gq"], -1.0), dk=one(s["gk"], -1.0))
    return out


def _exact_append(s, case):
    kp, vp = s["k_pages"].double(), s["v_pages"].double()
    q, row = s["q"].double(), 0
    table = s["page_table"].tolist()
    for i, (c, n) in enumerate(zip(_chunks(case), _lengths(case))):
        for p in range(n - c, n):
            k = s["k"][row].double()
            if case["rotary"]:
                k, q[row] = (_exact_rotate(x, p * s["frequencies"], case["interleaved"]) for x in (k, s["q"][row]))
            page, at = table[i][p // case["page"]], p % case["page"]
            kp[page, :, at], vp[page, :, at] = k, s["v"][row].double()
            row += 1
    return dict(k_pages=kp, v_pages=vp, **({"q": q} if case["rotary"] else {}))


def _exact_attention(s, case):
    Hq, Hkv, D, ps = case["Hq"], case["Hkv"], case["D"], case["page"]
    out, lse, row = [], [], 0
    for i, (c, n) in enumerate(zip(_chunks(case), _lengths(case))):
        pages = s["page_table"][i, : -(-n // ps)].long()
        heads = []
        for h in range(Hkv):
            k, v = (s[w][pages, h].reshape(-1, D)[:n].double() for w in ("k_pages", "v_pages"))
            for j in range(h * (Hq // Hkv), (h + 1) * (Hq // Hkv)):
                x = s["q"][row: row + c, j].double() @ k.T / math.sqrt(D)
                if case["causal"]:
                    x += torch.full((c, n), -math.inf, dtype=torch.float64, device=x.device).triu(n - c + 1)
                z = torch.logsumexp(x, -1)
                heads.append((torch.exp(x - z[:, None]) @ v, z))
        out.append(torch.stack([o for o, _ in heads], 1))
        lse.append(torch.stack([z for _, z in heads], 1))
        row += c
    return (torch.cat(out), torch.cat(lse)) if case["lse"] else torch.cat(out)


def _exact_pool(s, case):
    """The same steps one page at a time, over lists."""
    ps = case["page"]
    table, lens, refs = s["page_table"].tolist(), s["seq_lens"].tolist(), s["ref_counts"].tolist()
    pages = s["pages_"].clone()
    if case["op"] == "compact":
        count = sum(r > 0 for r in refs)
        holes = [p for p in range(count) if refs[p] == 0]
        for p in [p for p in range(count, len(refs)) if refs[p] > 0]:
            to = holes.pop(0)
            pages[:, :, to] = pages[:, :, p]
        return pages.double(), None, None, None
    for d in s["dst"].tolist():
        for p in table[d]:
            if p >= 0:
                refs[p] -= 1
        table[d], lens[d] = [-1] * len(table[d]), 0
    for a, d in zip(s["src"].tolist(), s["dst"].tolist()):
        table[d], lens[d] = list(table[a]), lens[a]
        if lens[a] % ps:
            to = refs.index(0)
            old, table[d][lens[a] // ps] = table[d][lens[a] // ps], to
            pages[:, :, to] = pages[:, :, old]
        for p in table[d]:
            if p >= 0:
                refs[p] += 1
    return pages.double(), None, None, None


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(s)
    if case["op"] == "append":
        return _exact_append(s, case)
    if case["op"] == "attention":
        return _exact_attention(s, case)
    return _exact_pool(s, case)
