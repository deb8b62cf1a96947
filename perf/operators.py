"""Operators of serving with a cache in pages and drafted tokens, as cases: what they are given, their plain form, and the calls of this package.

  append   keys and values of new tokens to the pages of a cache, 8-bit codes with one scale per row and head, or 16-bit values
  read     rows of such pages back as ordinary values
  attend   attention of the new tokens of every sequence over its pages
  probs    probabilities from logits, with a temperature per row
  verify   drafted tokens against the target's probabilities, from given random numbers

A step of a server that decodes with drafts runs append, attend, probs and verify one after the other.

The sequences of a case have different lengths, spread between `lo` and `hi` by a fixed rule, so that a case alone says how much work it is; the
values and the order of the pages come from the seed.
"""
import ctypes
import importlib.util
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8, "e4m3": torch.float8_e4m3fn}
CODE = {"f32": 0, "f16": 1, "bf16": 30, "i8": 24, "e4m3": 259}        # the package's type codes
TOP = {"i8": 127.0, "e4m3": 448.0}
TINY = 2.0 ** -100                                                     # rows of smaller values are stored as zeros
GOLDEN = 0.6180339887498949


def size(kind):
    return torch.empty(0, dtype=TORCH[kind]).element_size()


# ---- the cases -----------------------------------------------------------------------------

def paged(name, do, seqs, new, lo, hi, kv_heads, dim, kind, page, **more):
    c = dict(do=do, seqs=seqs, new=new, lo=lo, hi=hi, kv_heads=kv_heads, dim=dim, kind=kind, page=page, **more)
    return dict(c, name=name) if name else c


def append(name, *args, given="f32", rotated=True):
    return paged(name, "append", *args, given=given, rotated=rotated)


def read(name, *args, out="bf16"):
    return paged(name, "read", *args, out=out)


def attend(name, *args, heads, given="f32", out="bf16", window=0, sink=False, rotated=True):
    return paged(name, "attend", *args, heads=heads, given=given, out=out, window=window, sink=sink, rotated=rotated)


def probs(name, rows, vocab, temperature):
    c = dict(do="probs", rows=rows, vocab=vocab, temperature=temperature)
    return dict(c, name=name) if name else c


def verify(name, seqs, drafts, vocab, certain=False):
    c = dict(do="verify", seqs=seqs, drafts=drafts, vocab=vocab, certain=certain)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token of one sequence: what every decoding step adds to a layer's cache, bound by latency
        append("append-token", 1, 1, 700, 700, 8, 128, "e4m3", 16),
        # prompts of eight sequences on their way into an 8-bit cache
        append("append-prompts-i8", 8, 2048, 2048, 4096, 8, 128, "i8", 64),
        # one conversation of the 7B geometry read back for a snapshot
        read("read-7b", 1, 1, 1531, 1531, 32, 128, "i8", 16, out="f16"),
        # the caches of eight long conversations moved to 16 bits
        read("read-long", 8, 1, 3000, 20000, 8, 128, "e4m3", 64, out="bf16"),
        # a token of one conversation of the 7B geometry: f16 cache, f32 in and out, bound by latency
        attend("attend-token-7b", 1, 1, 521, 521, 32, 128, "f16", 16, heads=32, out="f32", rotated=False),
        # one token of each of 64 running sequences over an 8-bit cache
        attend("attend-64-i8", 64, 1, 500, 8192, 8, 128, "i8", 64, heads=32),
        # 16 sequences with up to five drafted tokens each, a window and sinks
        attend("attend-drafts-e4m3", 16, 6, 200, 6000, 8, 128, "e4m3", 32, heads=32, window=4096, sink=True),
        # the next 2048 tokens of two long documents
        attend("attend-prompts", 2, 2048, 9001, 16384, 8, 128, "bf16", 128, heads=32, given="bf16"),
        # the five rows of one sequence with four drafts
        probs("probs-5", 5, 32000, 0.8),
        # the rows of 64 sequences with seven drafts each, a larger vocabulary
        probs("probs-512", 512, 128000, 0.7),
        # four drafts of one sequence
        verify("verify-1", 1, 4, 32000),
        # up to seven drafts of each of 64 sequences
        verify("verify-64", 64, 7, 128000),
    ]


def draw(rng):
    def between(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    do = rng.choice(["append", "read", "attend", "attend", "attend", "attend", "probs", "verify"])
    if do == "probs":
        rows = between(1, 512)
        return probs(None, rows, between(1000, min(200000, 512 * 128000 // rows)), rng.choice([0.0, 0.6, 0.8, 1.0, 1.3]))
    if do == "verify":
        return verify(None, between(1, 64), rng.randint(0, 7), between(1000, 128000), certain=rng.random() < 0.25)
    group, kv_heads = rng.choice([(1, 8), (1, 32), (1, 40), (4, 2), (4, 4), (4, 8), (8, 4), (5, 3), (7, 1)])
    dim, page, kind = rng.choice([64, 80, 128, 128, 128]), rng.choice([8, 16, 20, 32, 64, 128]), rng.choice(["f16", "bf16", "i8", "e4m3"])
    shape = (kv_heads, dim, kind, page)
    if do == "append":
        seqs = between(1, 16)
        new = between(1, 16384 * 1024 // (seqs * kv_heads * dim))
        return append(None, seqs, new, new, new + between(1, 3000), *shape, given=rng.choice(["f32", "bf16", "f16"]), rotated=rng.random() < 0.7)
    if do == "read":
        seqs = between(1, 16)
        hi = between(1, 65536 * 1024 // (seqs * kv_heads * dim))
        return read(None, seqs, 1, max(1, hi // 3), hi, *shape, out=rng.choice(["f32", "bf16", "f16"]))
    window, sink, rotated, given = rng.choice([0, 0, 0, between(16, 4096)]), rng.random() < 0.3, rng.random() < 0.7, rng.choice(["f32", "bf16"])
    out = rng.choice(["bf16", "bf16", "f16", "f32"])
    more = dict(heads=group * kv_heads, given=given, out=out, window=window, sink=sink, rotated=rotated)
    role = rng.choice(["token", "tokens", "drafts", "prompt", "prompts"])
    if role in ("token", "tokens"):
        seqs = 1 if role == "token" else between(2, 64)
        hi = between(10, min(16384, 16 * 2 ** 20 * 32 // (seqs * kv_heads * dim)))
        return attend(None, seqs, 1, max(1, hi // 4), hi, *shape, **more)
    if role == "drafts":
        seqs, new = between(1, 32), rng.randint(2, 9)
        hi = between(20, min(16384, 8 * 2 ** 20 * 32 // (seqs * kv_heads * dim)))
        return attend(None, seqs, new, max(new, hi // 4), hi, *shape, **more)
    seqs = 1 if role == "prompt" else rng.randint(2, 6)
    new = between(20, 2048)
    most = 128 * 2 ** 30 // (seqs * group * kv_heads * new * dim)             # (products of one kind in the whole case)
    hi = between(new, max(new, min(16384, most)))
    return attend(None, seqs, new, max(new, hi // 2), hi, *shape, **more)


def spread(lo, hi, n, at):
    """n whole numbers from lo to hi, hi among them."""
    return [hi if s == 0 else lo + int((hi - lo) * ((s * GOLDEN + at) % 1.0)) for s in range(n)]


def lengths(case):
    """(positions, new tokens) of each sequence."""
    lens = spread(case["lo"], case["hi"], case["seqs"], 0.1)
    return lens, [min(n, m) for n, m in zip(spread((case["new"] + 1) // 2, case["new"], case["seqs"], 0.7), lens)]


def drafts_of(case):
    return spread(case["drafts"] // 2, case["drafts"], case["seqs"], 0.3)


def work(case):
    do = case["do"]
    if do == "probs":
        n = case["rows"] * case["vocab"]
        return {"bytes": 8 * n, "flops": 4 * n}
    if do == "verify":
        rows = case["seqs"] * case["vocab"] * (1 if case["certain"] else 2)          # the row that a token is drawn from, and the draft's
        return {"bytes": 4 * rows + 20 * sum(drafts_of(case)), "flops": 3 * rows}
    (lens, new), H, D = lengths(case), case["kv_heads"], case["dim"]
    row = H * (D * size(case["kind"]) + (4 if case["kind"] in TOP else 0)) * 2
    if do == "append":
        n = sum(new)
        return {"bytes": n * (row + 2 * H * D * size(case["given"]) + (D * 4 if case["rotated"] else 0)), "flops": n * H * D * 2 * 6}
    if do == "read":
        return {"bytes": sum(lens) * (row + 2 * H * D * size(case["out"])), "flops": 2 * sum(lens) * H * D}
    w, pairs, seen = case["window"], 0, 0
    for n, m in zip(lens, new):
        first = n - m                                                   # positions first .. n - 1 ask
        reach = w or n
        full = max(0, n - max(first, reach))                            # those that see `reach` keys
        pairs += full * reach + sum(p + 1 for p in range(first, n - full))
        seen += n - max(0, first + 1 - reach)
    return {"bytes": seen * row + sum(new) * case["heads"] * D * (size(case["given"]) + size(case["out"])), "flops": 4 * pairs * case["heads"] * D}


# ---- inputs --------------------------------------------------------------------------------

def rotations(gen, tokens, dim):
    """{cos, sin} of the angles of `tokens` positions, as a rotary table has them."""
    at = torch.randint(0, 16384, (tokens, 1), generator=gen, device="cuda").double()
    angle = at * 10000.0 ** (-torch.arange(dim // 2, device="cuda").double() / (dim // 2))
    return torch.stack([angle.cos(), angle.sin()], -1).float().reshape(tokens, dim).contiguous()


def quantised(x, kind):
    """(codes, scale of each row of the last axis) of f32 values."""
    top = x.abs().amax(-1, keepdim=True)
    full = torch.full_like(top, TOP[kind])
    fine = top < math.inf
    live = fine & (top >= TINY)
    scale = torch.where(live, top / full, torch.where(fine, 0.0, math.nan))
    code = x * torch.where(live, full / torch.where(live, top, 1.0), 0.0)
    code = torch.where(live, code, 0.0)
    return (code.round() if kind == "i8" else code).to(TORCH[kind]), scale.squeeze(-1)


def pages(gen, case, lens, filled):
    """A pool of pages in any order, with the table of every sequence's pages."""
    H, D, R, kind = case["kv_heads"], case["dim"], case["page"], case["kind"]
    counts = [-(-n // R) for n in lens]
    width, total = max(counts), sum(counts)
    order = torch.randperm(total + 3, generator=gen, device="cuda")[:total].to(torch.int32)
    table = torch.zeros(len(lens), width, dtype=torch.int32, device="cuda")
    mine = torch.arange(width, device="cuda")[None] < torch.tensor(counts, device="cuda")[:, None]
    table[mine] = order
    state = {"table": table}
    for name in "kv":
        if not filled:
            state[name] = torch.zeros(total + 3, H, R, D, dtype=TORCH[kind], device="cuda")
            if kind in TOP:
                state[name + "_scale"] = torch.zeros(total + 3, H, R, device="cuda")
            continue
        x = torch.randn(total + 3, H, R, D, generator=gen, device="cuda")
        x *= torch.rand(total + 3, H, R, 1, generator=gen, device="cuda") + 0.5          # (rows differ in size, as a model's do)
        if kind in TOP:
            state[name], state[name + "_scale"] = quantised(x, kind)
        else:
            state[name] = x.to(TORCH[kind])
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    do, state = case["do"], {"case": case}

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    if do == "probs":
        state["logits"] = 3.0 * normal(case["rows"], case["vocab"])
        state["temperature"] = torch.full((case["rows"],), case["temperature"], device="cuda")
        state["out"] = torch.empty_like(state["logits"])
    elif do == "verify":
        n = drafts_of(case)
        starts = [sum(n[:s]) + s for s in range(len(n) + 1)]
        rows, vocab = starts[-1], case["vocab"]
        logits = 3.0 * normal(rows, vocab)
        state["target"] = torch.softmax(logits, -1)
        state["draft"] = torch.softmax(logits + 0.5 * normal(rows, vocab), -1)
        state["drafted"] = torch.multinomial(state["draft"], 1, generator=gen).squeeze(1).to(torch.int32)
        if case["certain"]:
            state["draft"] = None
        state["accept"], state["pick"] = uniform(rows), uniform(len(n))
        state["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        state["tokens"], state["accepted"] = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(len(n), dtype=torch.int32, device="cuda")
        state["most"] = case["drafts"] + 1
    else:
        lens, new = lengths(case)
        state |= pages(gen, case, lens, filled=do != "append")
        state["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        state["starts"] = torch.tensor([sum(new[:s]) for s in range(len(new) + 1)], dtype=torch.int32, device="cuda")
        tokens, H, D = sum(new), case["kv_heads"], case["dim"]
        state["most"] = max(new)
        if do == "append":
            state["new_k"], state["new_v"] = (normal(tokens, H * D).to(TORCH[case["given"]]) for _ in range(2))
        elif do == "read":
            state["out_k"], state["out_v"] = (torch.zeros(len(lens), H, max(lens), D, dtype=TORCH[case["out"]], device="cuda") for _ in range(2))
        else:
            state["q"] = (1.5 * normal(tokens, case["heads"] * D)).to(TORCH[case["given"]])
            state["out"] = torch.empty(tokens, case["heads"] * D, dtype=TORCH[case["out"]], device="cuda")
            state["sink"] = normal(case["heads"]) if case["sink"] else None
        if do != "read":
            state["angles"] = rotations(gen, tokens, D) if case["rotated"] else None
    torch.cuda.synchronize()
    return state


# ---- the plain form --------------------------------------------------------------------------

def rotated(x, angles):
    """x [tokens][heads][dim]: pairs of neighbours turned by the angles of their token."""
    if angles is None:
        return x
    c, s = angles[:, None, 0::2], angles[:, None, 1::2]
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)


def owners(state, tokens):
    """The sequence of every token, and its position there."""
    row = torch.arange(tokens, device="cuda")
    starts, lens = state["starts"].long(), state["lens"].long()
    seq = torch.searchsorted(starts[1:], row, right=True)
    return seq, lens[seq] - starts[seq + 1] + row


def plain_append(state):
    case = state["case"]
    H, D, R, tokens = case["kv_heads"], case["dim"], case["page"], state["new_k"].shape[0]
    seq, at = owners(state, tokens)
    page, row = state["table"][seq, at // R].long(), at % R
    for name in "kv":
        x = state["new_" + name].float().view(tokens, H, D)
        x = rotated(x, state["angles"]) if name == "k" else x
        if case["kind"] in TOP:
            x, scale = quantised(x, case["kind"])
            state[name + "_scale"][page, :, row] = scale
        state[name].view(torch.uint8)[page, :, row] = x.to(TORCH[case["kind"]]).view(torch.uint8)
    return written(state)


def written(state):
    """The whole cache: 16-bit values, or the codes (as numbers) with their scales."""
    return {n: state[n] for n in ("k", "v", "k_scale", "v_scale") if n in state}


def unpacked(state, name):
    """f32 values [sequences][heads][positions of the table][dim]"""
    x = state[name][state["table"].long()].float()
    if name + "_scale" in state:
        x = x * state[name + "_scale"][state["table"].long()][..., None]
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3)


def plain_read(state):
    for name in "kv":
        out = state["out_" + name]
        x = unpacked(state, name)[:, :, :out.shape[2]]
        there = torch.arange(out.shape[2], device="cuda") < state["lens"][:, None]
        out.copy_(torch.where(there[:, None, :, None], x, out.float()))
    return state["out_k"], state["out_v"]


def plain_attend(state):
    case, out = state["case"], state["out"]
    H, D, tokens = case["kv_heads"], case["dim"], out.shape[0]
    G, starts, lens = case["heads"] // H, state["starts"].long(), state["lens"].long()
    q = rotated(state["q"].float().view(tokens, case["heads"], D), state["angles"])
    i = torch.arange(state["most"], device="cuda")
    row = starts[:-1, None] + i                                         # [sequences][new]
    live = row < starts[1:, None]
    row = row.clamp(max=tokens - 1)
    at = lens[:, None] - starts[1:, None] + row
    k = unpacked(state, "k")
    q = q[row].view(*row.shape, H, G, D).permute(0, 2, 3, 1, 4).flatten(2, 3)
    s = (q @ k.mT).view(len(lens), H, G, len(i), -1).mul_(D ** -0.5)
    del k
    j = torch.arange(s.shape[-1], device="cuda")
    hidden = j > at[..., None]
    if case["window"]:
        hidden |= j <= at[..., None] - case["window"]
    s.masked_fill_(hidden[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    sink = state["sink"]
    if sink is not None:
        sink = sink.view(H, G, 1, 1)
        top = torch.maximum(top, sink)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    if sink is not None:
        total = total + (sink - top).exp()
    x = (p.flatten(2, 3) @ unpacked(state, "v")).view(len(lens), H, G, len(i), D) / total
    x = x.permute(0, 3, 1, 2, 4).flatten(2)
    out[row[live]] = x[live].to(out.dtype)
    return out


def plain_probs(state):
    x = state["logits"]
    if state["case"]["temperature"] == 0.0:
        first = x.argmax(-1, keepdim=True)
        return torch.zeros_like(x).scatter_(1, first, 1.0)
    x = x / state["temperature"][:, None]
    e = (x - x.amax(-1, keepdim=True)).exp()
    return e / e.sum(-1, keepdim=True)


def plain_verify(state):
    p, q, starts = state["target"], state["draft"], state["starts"].long()
    n, first = starts[1:] - starts[:-1] - 1, starts[:-1]
    i = torch.arange(state["most"], device="cuda")
    row = (first[:, None] + i).clamp(max=p.shape[0] - 1)
    token = state["drafted"][row].long()
    mine = p[row, token].double()
    theirs = torch.ones_like(mine) if q is None else q[row, token].double()
    good = (state["accept"][row].double() * theirs < mine) & (i < n[:, None])
    accepted = good.long().cumprod(-1).sum(-1)
    at = first + accepted
    rejected = (accepted < n)[:, None]
    target = p[at].double()
    guess = torch.zeros_like(target).scatter_(1, state["drafted"][at].long()[:, None], 1.0) if q is None else q[at].double()
    rest = torch.where(rejected, (target - guess).clamp(min=0.0), target)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, target)
    mass = rest.cumsum(-1)
    past = mass > state["pick"].double()[:, None] * mass[:, -1:]
    drawn = past.int().argmax(-1)
    tokens = torch.full_like(state["tokens"], -1)
    inside = (i < accepted[:, None])
    tokens[row[inside]] = state["drafted"][row[inside]]
    tokens[at] = drawn.to(torch.int32)
    return tokens, accepted.to(torch.int32)


# ---- the package's calls -----------------------------------------------------------------------

def package():
    """The package directory has a hyphen in its name."""
    name = "llama_vulkan_b200"
    if name not in sys.modules:
        at = os.path.join(ROOT, "llama-vulkan_b200")
        spec = importlib.util.spec_from_file_location(name, os.path.join(at, "__init__.py"), submodule_search_locations=[at])
        sys.modules[name] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[name])
    return sys.modules[name]


def context():
    """A program has one context for its GPU."""
    pkg = package()
    if not hasattr(pkg, "operators_context"):
        pkg.operators_context = pkg.Context(0)
    return pkg, pkg.operators_context


def at(t):
    return None if t is None else t.data_ptr()


def described(state):
    """The argument blocks and the workspace of a state's call, made once: a program keeps them from step to step."""
    pkg, ctx = context()
    case, do = state["case"], state["case"]["do"]
    if do == "verify":
        a = pkg.VerifyArgs(target=at(state["target"]), target_ld=case["vocab"], draft=at(state["draft"]), draft_ld=case["vocab"], vocab=case["vocab"],
                           drafted=at(state["drafted"]), starts=at(state["starts"]), seqs=case["seqs"], rows=state["target"].shape[0],
                           accept=at(state["accept"]), pick=at(state["pick"]), tokens=at(state["tokens"]), accepted=at(state["accepted"]))
        return a, None
    c = pkg.PagedCache(k=at(state["k"]), v=at(state["v"]), k_scale=at(state.get("k_scale")), v_scale=at(state.get("v_scale")), type=CODE[case["kind"]],
                       pages=state["k"].shape[0], page_rows=case["page"], kv_heads=case["kv_heads"], dim=case["dim"], table=at(state["table"]),
                       table_ld=state["table"].shape[1], lens=at(state["lens"]), starts=at(state["starts"]), seqs=case["seqs"])
    if do != "attend":
        return c, None
    a = pkg.PagedAttentionArgs(cache=c, q=at(state["q"]), q_type=CODE[case["given"]], q_ld=state["q"].shape[1], heads=case["heads"], tokens=state["q"].shape[0],
                               max_new=state["most"], max_len=case["hi"], scale=case["dim"] ** -0.5, window=case["window"], sink=at(state["sink"]),
                               angles=at(state["angles"]), angle_ld=case["dim"], angle_pairs=case["dim"] // 2 if case["rotated"] else 0,
                               out=at(state["out"]), out_type=CODE[case["out"]], out_ld=state["out"].shape[1])
    scratch = torch.empty(max(16, ctx.lib.lv_paged_attention_scratch_bytes(ctx.handle, ctypes.byref(a))), dtype=torch.uint8, device="cuda")
    return a, scratch


def run_own(state):
    pkg, ctx = context()
    case, do, lib = state["case"], state["case"]["do"], ctx.lib
    if do == "probs":
        rows, vocab = state["logits"].shape
        pkg.check(lib.lv_probabilities(ctx.handle, at(state["out"]), vocab, at(state["logits"]), vocab, vocab, rows, at(state["temperature"])))
        return state["out"]
    if "described" not in state:
        state["described"] = described(state)
    a, scratch = state["described"]
    if do == "verify":
        pkg.check(lib.lv_verify_drafts(ctx.handle, ctypes.byref(a)))
        return state["tokens"], state["accepted"]
    if do == "append":
        tokens, width = state["new_k"].shape
        pkg.check(lib.lv_paged_append(ctx.handle, ctypes.byref(a), at(state["new_k"]), at(state["new_v"]), CODE[case["given"]], width, at(state["angles"]),
                                      case["dim"], case["dim"] // 2 if case["rotated"] else 0, tokens))
        return written(state)
    if do == "read":
        _, heads, rows, dim = state["out_k"].shape
        pkg.check(lib.lv_paged_read(ctx.handle, ctypes.byref(a), at(state["out_k"]), at(state["out_v"]), CODE[case["out"]], heads * rows * dim, rows * dim, dim,
                                    0, rows))
        return state["out_k"], state["out_v"]
    pkg.check(lib.lv_paged_attention(ctx.handle, ctypes.byref(a), scratch.data_ptr(), scratch.numel()))
    return state["out"]


def run(state):
    if own:
        return run_own(state)
    return {"append": plain_append, "read": plain_read, "attend": plain_attend, "probs": plain_probs, "verify": plain_verify}[state["case"]["do"]](state)


# ---- in 64 bits ---------------------------------------------------------------------------------

def exact(case, seed):
    """From the definitions, a sequence at a time.  Codes and tokens are whole numbers and have no value between them."""
    do = case["do"]
    if do == "verify":
        return None
    s = prepare(case, seed)
    if do == "probs":
        x = s["logits"].double()
        if case["temperature"] == 0.0:
            hot = torch.zeros_like(x)
            hot[torch.arange(len(x)), x.max(1).indices] = 1.0
            return hot
        return torch.softmax(x / s["temperature"].double()[:, None], 1)
    H, D, R, kind = case["kv_heads"], case["dim"], case["page"], case["kind"]
    lens, new = lengths(case)
    if do == "append":
        got = {n: s[n].double() for n in written(s)}
        before = 0
        for seq, (n, m) in enumerate(zip(lens, new)):
            for name in "kv":
                x = s["new_" + name][before:before + m].double().view(m, H, D)
                if name == "k" and case["rotated"]:
                    turn = torch.view_as_complex(s["angles"][before:before + m].double().view(m, 1, D // 2, 2))
                    x = torch.view_as_real(torch.view_as_complex(x.reshape(m, H, D // 2, 2)) * turn).reshape(m, H, D)
                where = torch.arange(n - m, n, device="cuda")
                page = s["table"][seq].long()[where // R]
                if kind in TOP:
                    got[name + "_scale"][page, :, where % R] = x.abs().max(-1).values / TOP[kind]
                else:
                    got[name][page, :, where % R] = x
            before += m
        if kind in TOP:
            got["k"] = got["v"] = None
        return got

    def sequence(name, seq):
        """[heads][positions][dim]"""
        page = s["table"][seq, :-(-lens[seq] // R)].long()
        x = s[name][page].double()
        if kind in TOP:
            x = x * s[name + "_scale"][page].double().unsqueeze(-1)
        return x.transpose(0, 1).reshape(H, -1, D)[:, :lens[seq]]

    if do == "read":
        outs = []
        for name in "kv":
            out = torch.zeros(len(lens), H, max(lens), D, dtype=torch.float64, device="cuda")
            for seq, n in enumerate(lens):
                out[seq, :, :n] = sequence(name, seq)
            outs.append(out)
        return outs
    out, before, G = torch.empty(sum(new), case["heads"], D, dtype=torch.float64, device="cuda"), 0, case["heads"] // H
    for seq, (n, m) in enumerate(zip(lens, new)):
        q = s["q"][before:before + m].double().view(m, case["heads"], D)
        if case["rotated"]:
            turn = torch.view_as_complex(s["angles"][before:before + m].double().view(m, 1, D // 2, 2))
            q = torch.view_as_real(torch.view_as_complex(q.reshape(m, -1, D // 2, 2)) * turn).reshape(m, -1, D)
        k, v = sequence("k", seq), sequence("v", seq)
        here, there = torch.arange(n - m, n, device="cuda")[:, None], torch.arange(n, device="cuda")
        seen = (there <= here) & ((there > here - case["window"]) if case["window"] else True)
        for h in range(case["heads"]):
            z = (q[:, h] @ k[h // G].T / math.sqrt(D)).masked_fill(~seen, -math.inf)
            if case["sink"]:
                z = torch.cat([z, s["sink"][h].double().expand(m, 1)], 1)
            out[before:before + m, h] = torch.softmax(z, 1)[:, :n] @ v[h // G]
        before += m
    return out.flatten(1)
