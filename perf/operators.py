"""Cases of the decoding operators: rotary positions, the paged key-value cache,
attention of one new token over that cache.

A protein language model beside the pair stack generates or scores a sequence
token by token: queries and keys are rotated by their positions, keys and
values enter a cache kept in pages (as they are, or in 8 bits with a scale per
row), and each new token attends to its sequence's pages.  Every case is one
such call; ``listed()`` names the fixed ones, ``draw()`` gives others of the
same ranges.

A case is a dict of plain values:

  op         "rotary" | "cache" | "attention"
  batch      sequences of the call
  dtype      "f32" | "f16" | "bf16": queries, and keys and values as computed
  head_dim   channels of a head

rotary:      tokens per sequence, q_heads, k_heads, rotary_dim (the rotated
             part of the head), layout "half" | "interleaved", factor (context
             scaling, 1: none), scaling "linear" | "by_parts", max_position,
             direction "forward" | "train" (outputs, then both gradients)
cache:       heads, page (slots a page), context (tokens each sequence holds),
             new (tokens written to each), format (the cache's type: "f32" |
             "f16" | "bf16" | "fp8" | "int8"), read "new" | "all" (rows read
             back after the write; a plain cache returns itself as well)
attention:   q_heads, heads, page, shortest and longest (lengths are spread
             evenly between them), format, window (0: all keys)

The plain forms compute in 32 bits (angles in 64) with elementary torch
operations and round once at the end.
"""
from __future__ import annotations

import math
import random

import torch

own = False
DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
FORMATS = {**DTYPES, "fp8": torch.float8_e4m3fn, "int8": torch.int8}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "fp8": 1, "int8": 1}
BASE = 10000.0
ORIGINAL = 4096      # context a scaled model was trained for
SLOW, FAST = 1.0, 32.0


def listed():
    return [
        # one decoding step of 64 sequences far into a scaled context: latency
        dict(name="rotary_step", op="rotary", batch=64, tokens=1, q_heads=32, k_heads=8,
             head_dim=128, rotary_dim=128, layout="half", factor=32.0, scaling="by_parts",
             max_position=131072, dtype="bf16", direction="forward"),
        # a batch of prompts, shared key heads
        dict(name="rotary_prompt", op="rotary", batch=4, tokens=4096, q_heads=32, k_heads=8,
             head_dim=128, rotary_dim=128, layout="half", factor=1.0, scaling="linear",
             max_position=4096, dtype="bf16", direction="forward"),
        # training on odd lengths, positions in a part of the head, FP32
        dict(name="rotary_train", op="rotary", batch=3, tokens=1021, q_heads=16, k_heads=16,
             head_dim=80, rotary_dim=32, layout="interleaved", factor=4.0, scaling="linear",
             max_position=16384, dtype="f32", direction="train"),
        # the new tokens of 64 sequences enter a plain cache
        dict(name="cache_step_bf16", op="cache", batch=64, context=511, new=1, heads=8,
             head_dim=128, page=16, dtype="bf16", format="bf16", read="new"),
        # the next chunk of two long prompts enters an FP8 cache, and the
        # whole context comes back for the chunk's own attention
        dict(name="cache_chunk_fp8", op="cache", batch=2, context=30001, new=2048, heads=8,
             head_dim=128, page=64, dtype="bf16", format="fp8", read="all"),
        # prompts of odd length into an INT8 cache, read back
        dict(name="cache_prompt_int8", op="cache", batch=5, context=0, new=1537, heads=16,
             head_dim=64, page=32, dtype="f16", format="int8", read="all"),
        # one short sequence, the pair stack's heads in FP32: latency
        dict(name="attention_short_f32", op="attention", batch=1, shortest=124, longest=124,
             q_heads=4, heads=4, head_dim=32, page=16, dtype="f32", format="f32", window=0),
        # an ordinary serving batch of ragged lengths, grouped heads
        dict(name="attention_ragged_bf16", op="attention", batch=32, shortest=1, longest=4097,
             q_heads=32, heads=8, head_dim=128, page=16, dtype="bf16", format="bf16", window=0),
        # one very long sequence: the length itself has to be split
        dict(name="attention_long_bf16", op="attention", batch=1, shortest=131071,
             longest=131071, q_heads=32, heads=8, head_dim=128, page=64, dtype="bf16",
             format="bf16", window=0),
        # a large batch of long sequences in an FP8 cache
        dict(name="attention_batch_fp8", op="attention", batch=16, shortest=20001,
             longest=65536, q_heads=64, heads=8, head_dim=128, page=64, dtype="bf16",
             format="fp8", window=0),
        # local attention, a head of its own per query head, INT8 cache
        dict(name="attention_window_int8", op="attention", batch=24, shortest=300,
             longest=9001, q_heads=16, heads=16, head_dim=64, page=32, dtype="f16",
             format="int8", window=1000),
        # wide heads shared by all queries, FP32 throughout
        dict(name="attention_wide_f32", op="attention", batch=7, shortest=513, longest=8190,
             q_heads=24, heads=2, head_dim=256, page=128, dtype="f32", format="f32", window=0),
    ]


def draw(rng):
    def size(lo, hi):  # spread over the logarithm
        return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))

    op = rng.choice(["rotary", "cache", "attention", "attention"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    if op == "rotary":
        head_dim = rng.choice([32, 64, 80, 96, 128, 256])
        rotary_dim = rng.choice([head_dim, head_dim, head_dim // 2,
                                 2 * rng.randint(1, head_dim // 2)])
        k_heads = rng.choice([1, 2, 4, 8, 16])
        q_heads = k_heads * rng.choice([1, 2, 4, 5])
        batch = size(1, 64)
        room = 16384 * 40 * 128 // ((q_heads + k_heads) * head_dim * batch)
        tokens = size(1, max(1, min(8192, room // (2 if dtype == "f32" else 1))))
        direction = rng.choice(["forward", "forward", "train"])
        if direction == "train":
            tokens = max(1, tokens // 2)
        factor = rng.choice([1.0, 2.0, 8.0, 32.0])
        return dict(op=op, batch=batch, tokens=tokens, q_heads=q_heads, k_heads=k_heads,
                    head_dim=head_dim, rotary_dim=rotary_dim,
                    layout=rng.choice(["half", "interleaved"]), factor=factor,
                    scaling=rng.choice(["linear", "by_parts"]),
                    max_position=max(tokens, size(64, 1 << 20)), dtype=dtype,
                    direction=direction)
    head_dim = rng.choice([32, 64, 128, 128, 256])
    page = rng.choice([16, 32, 64, 128, 256])
    heads = rng.choice([1, 2, 4, 8, 16])
    form = rng.choice([dtype, "fp8", "int8"])
    batch = size(1, 64)
    if op == "cache":
        # at most the listed chunk's 64 K rows of 8 heads of 128
        total = 65536 * 8 * 128 // (heads * head_dim * batch)
        new = size(1, max(1, min(4096, total // (8 if dtype == "f32" else 4))))
        context = rng.choice([0, size(1, max(1, min(65536, total // 2)))])
        read = rng.choice(["new", "all"])
        return dict(op=op, batch=batch, context=context, new=new, heads=heads,
                    head_dim=head_dim, page=page, dtype=dtype, format=form, read=read)
    group = rng.choice([1, 2, 4, 5, 8, 16, 24])
    total = 16 * 40000 * 8 * 128 // (heads * head_dim * batch * max(1, group // 8))
    longest = size(1, max(1, min(131072, total // BYTES[form])))
    shortest = rng.choice([longest, max(0, rng.randint(0, longest)), 0])
    window = rng.choice([0, 0, 0, size(1, 4096)])
    return dict(op=op, batch=batch, shortest=shortest, longest=longest, q_heads=heads * group,
                heads=heads, head_dim=head_dim, page=page, dtype=dtype, format=form,
                window=window)


# ---------------------------------------------------------------- inputs

def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _randn(shape, g, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=DEVICE).to(dtype)


def _frequencies(case, dtype=torch.float64):
    """The rotation a position, in radians, of each pair; and the outputs' factor."""
    r, factor = case["rotary_dim"], case["factor"]
    i = torch.arange(r // 2, dtype=dtype, device=DEVICE)
    f = torch.pow(torch.tensor(BASE, dtype=dtype, device=DEVICE), -2.0 * i / r)
    if factor == 1.0:
        return f, 1.0
    if case["scaling"] == "linear":
        return f / factor, 1.0
    turns = ORIGINAL * f / (2.0 * math.pi)
    keep = ((turns - SLOW) / (FAST - SLOW)).clamp(0.0, 1.0)
    return f / factor * (1.0 - keep) + f * keep, 0.1 * math.log(factor) + 1.0


def _lengths(case):
    b, lo, hi = case["batch"], case["shortest"], case["longest"]
    return [hi - (hi - lo) * i // max(1, b - 1) for i in range(b)]


def _table(case, per_sequence, g):
    """Pages of each sequence, in the order of a pool long in use: any order."""
    pages = case["batch"] * per_sequence + 3
    order = torch.randperm(pages, generator=g, device=DEVICE)[:case["batch"] * per_sequence]
    return order.view(case["batch"], per_sequence).to(torch.int32), pages


def _quantise(x, form):
    """8-bit codes of the rows of x and their scales, in 32 bits."""
    x = x.float()
    top = x.abs().amax(-1, keepdim=True)
    if form == "fp8":  # the least power of two that brings the row within 448
        mantissa, exponent = torch.frexp(top)
        e = (exponent - 9 + (mantissa > 0.875).int()).clamp(min=-126)
        scale = torch.ldexp(torch.ones_like(top), e)
        codes = (x / scale).to(torch.float8_e4m3fn)
    else:
        scale = top * (1.0 / 127.0)
        codes = torch.round(x * torch.reciprocal(scale)).to(torch.int8)
    return codes, scale.squeeze(-1)


def _pool(case, pages, g, rows=1 << 16):
    """A cache's k and v (and scales): rows of unit variance, each with a gain of its own."""
    shape = (pages, case["heads"], case["page"], case["head_dim"])
    form = case["format"]
    out = []
    for _ in range(2):
        data = torch.empty(shape, dtype=FORMATS[form], device=DEVICE)
        scale = None
        if form in ("fp8", "int8"):
            scale = torch.empty(shape[:3], dtype=torch.float32, device=DEVICE)
        step = max(1, rows // (case["heads"] * case["page"]))
        for p in range(0, pages, step):
            part = (min(step, pages - p),) + shape[1:]
            gain = torch.exp(0.3 * torch.randn(part[:3], generator=g, device=DEVICE))
            x = _randn(part, g) * gain[..., None]
            if scale is None:
                data[p:p + step] = x.to(data.dtype)
            else:
                codes, scale[p:p + step] = _quantise(x, form)
                data.view(torch.int8)[p:p + step] = codes.view(torch.int8)
        out += [data, scale]
    return out


def _cache_of(k, k_scale, v, v_scale):
    if not own:
        return None
    from fireprot_amd import kv_cache

    return kv_cache.PagedCache(k, v, k_scale, v_scale)


def prepare(case, seed):
    g = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    b, d = case["batch"], case["head_dim"]
    state = {"case": case}
    if case["op"] == "rotary":
        n, hq, hk = case["tokens"], case["q_heads"], case["k_heads"]
        # q and k are columns of one fused projection's output
        fused = _randn((b, n, (hq + 2 * hk) * d), g, dtype)
        q = fused[..., :hq * d].view(b, n, hq, d)
        k = fused[..., hq * d:(hq + hk) * d].view(b, n, hk, d)
        start = torch.randint(0, case["max_position"] - n + 1, (b, 1), generator=g, device=DEVICE)
        state.update(q=q, k=k, positions=start + torch.arange(n, device=DEVICE))
        if case["direction"] == "train":
            state.update(gq=_randn(q.shape, g, dtype), gk=_randn(k.shape, g, dtype))
        if own:
            from fireprot_amd import rotary

            scaled = case["factor"] != 1.0
            state["frequencies"] = rotary.rotary_frequencies(
                case["rotary_dim"], base=BASE, scaling=case["scaling"] if scaled else None,
                factor=case["factor"], original_length=ORIGINAL, slow=SLOW, fast=FAST,
                device=DEVICE)
        else:
            state["frequencies"] = _frequencies(case)
        return state
    if case["op"] == "cache":
        length = case["context"] + case["new"]
        table, pages = _table(case, -(-length // case["page"]), g)
        k, k_scale, v, v_scale = _pool(case, pages, g)
        heads, new = case["heads"], case["new"]
        fused = _randn((b * new, (4 + 2) * heads, d), g)
        fused *= torch.exp(0.3 * torch.randn(fused.shape[:2], generator=g, device=DEVICE))[..., None]
        fused = fused.to(dtype)
        position = torch.arange(length, device=DEVICE)
        slots = (table[:, position // case["page"]].long() * case["page"]
                 + position % case["page"])
        written = slots[:, case["context"]:].clone()
        if new > 1:  # the last sequence's batch entry is padded: no slot
            written[-1, new - new // 8:] = -1
        read = written if case["read"] == "new" else slots
        state.update(k_new=fused[:, 4 * heads:5 * heads], v_new=fused[:, 5 * heads:],
                     k=k, v=v, k_scale=k_scale, v_scale=v_scale, written=written.reshape(-1),
                     read=read.reshape(-1), cache=_cache_of(k, k_scale, v, v_scale))
        return state
    table, pages = _table(case, max(1, -(-case["longest"] // case["page"])), g)
    k, k_scale, v, v_scale = _pool(case, pages, g)
    known = _lengths(case)
    random.Random(seed).shuffle(known)
    lengths = torch.tensor(known, dtype=torch.int32, device=DEVICE)
    # trained heads look at few keys: logits of standard deviation near 2
    q = _randn((b, case["q_heads"], d), g) * 2.0
    state.update(q=q.to(dtype), k=k, v=v, k_scale=k_scale, v_scale=v_scale, table=table,
                 lengths=lengths, known_lengths=known, scale=d ** -0.5, cache=_cache_of(k, k_scale, v, v_scale))
    return state


# ---------------------------------------------------------------- one pass

def _rotate(x, cos, sin, case):
    r = case["rotary_dim"]
    y = x.float().clone()
    if case["layout"] == "half":
        a, b = y[..., :r // 2].clone(), y[..., r // 2:r].clone()
        y[..., :r // 2], y[..., r // 2:r] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = y[..., 0:r:2].clone(), y[..., 1:r:2].clone()
        y[..., 0:r:2], y[..., 1:r:2] = a * cos - b * sin, b * cos + a * sin
    return y.to(x.dtype)


def _run_rotary(state):
    case = state["case"]
    if own:
        from fireprot_amd import rotary

        out = rotary.apply_rotary(state["q"], state["k"], state["positions"],
                                  state["frequencies"], layout=case["layout"])
        if case["direction"] == "forward":
            return out
        return *out, *rotary.rotary_backward(state["gq"], state["gk"], state["positions"],
                                             state["frequencies"], layout=case["layout"])
    frequencies, factor = state["frequencies"]
    angle = (state["positions"].double()[..., None] * frequencies)[:, :, None]
    cos, sin = (torch.cos(angle) * factor).float(), (torch.sin(angle) * factor).float()
    out = (_rotate(state["q"], cos, sin, case), _rotate(state["k"], cos, sin, case))
    if case["direction"] == "forward":
        return out
    return *out, _rotate(state["gq"], cos, -sin, case), _rotate(state["gk"], cos, -sin, case)


def _run_cache(state):
    case = state["case"]
    plain = case["format"] in DTYPES
    if own:
        from fireprot_amd import kv_cache

        kv_cache.cache_write(state["cache"], state["k_new"], state["v_new"], state["written"])
        rows = kv_cache.cache_read(state["cache"], state["read"], dtype=DTYPES[case["dtype"]])
    else:
        page = case["page"]
        kept = state["written"] >= 0
        slots = state["written"][kept]
        p, o = slots // page, slots % page
        for x, data, scale in ((state["k_new"], state["k"], state["k_scale"]),
                               (state["v_new"], state["v"], state["v_scale"])):
            if plain:
                data[p, :, o] = x[kept].to(data.dtype)
            else:
                codes, scale[p, :, o] = _quantise(x[kept], case["format"])
                data.view(torch.int8)[p, :, o] = codes.view(torch.int8)
        p, o = state["read"].clamp(min=0) // page, state["read"].clamp(min=0) % page
        rows = []
        for data, scale in ((state["k"], state["k_scale"]), (state["v"], state["v_scale"])):
            if plain:
                x = data[p, :, o].float()
            else:
                x = data.view(torch.int8)[p, :, o].view(data.dtype).float() * scale[p, :, o][..., None]
            x = torch.where((state["read"] >= 0)[:, None, None], x, 0.0)
            rows.append(x.to(DTYPES[case["dtype"]]))
    if plain:
        return rows[0], rows[1], state["k"], state["v"]
    return rows[0], rows[1], state["k_scale"], state["v_scale"]


def _attend(state, b, n):
    """Sequence b's output from its n keys."""
    case = state["case"]
    lo = max(0, n - case["window"]) if case["window"] else 0
    j = torch.arange(lo, n, device=DEVICE)
    p, o = state["table"][b, j // case["page"]].long(), j % case["page"]
    kv = []
    for data, scale in ((state["k"], state["k_scale"]), (state["v"], state["v_scale"])):
        if scale is None:
            x = data[p, :, o].float()
        else:
            x = data.view(torch.int8)[p, :, o].view(data.dtype).float()
            x *= scale[p, :, o][..., None]
        kv.append(x.transpose(0, 1).contiguous())  # [heads, n, d]
    q = state["q"][b].float().view(case["heads"], -1, case["head_dim"])
    s = torch.bmm(q, kv[0].transpose(1, 2).contiguous()) * state["scale"]
    top = s.amax(-1, keepdim=True)
    w = torch.exp(s - top)
    total = w.sum(-1, keepdim=True)
    o = torch.bmm(w, kv[1]) / total
    lse = top + torch.log(total)
    return o.reshape(case["q_heads"], -1), lse.reshape(-1)


def _run_attention(state):
    case = state["case"]
    if own:
        from fireprot_amd import paged_attention

        return paged_attention.paged_attention(
            state["q"], state["cache"], state["table"], state["lengths"], scale=state["scale"],
            window=case["window"], max_length=case["longest"], return_lse=True)
    out = torch.zeros(state["q"].shape, dtype=torch.float32, device=DEVICE)
    lse = torch.full(state["q"].shape[:2], float("-inf"), dtype=torch.float32, device=DEVICE)
    for b, n in enumerate(state["known_lengths"]):
        if n > 0:
            out[b], lse[b] = _attend(state, b, n)
    return out.to(state["q"].dtype), lse


def run(state):
    return {"rotary": _run_rotary, "cache": _run_cache,
            "attention": _run_attention}[state["case"]["op"]](state)


# ---------------------------------------------------------------- what a pass needs

def work(case):
    e, d, b = BYTES[case["dtype"]], case["head_dim"], case["batch"]
    if case["op"] == "rotary":
        rows = b * case["tokens"] * (case["q_heads"] + case["k_heads"])
        sides = 2 if case["direction"] == "train" else 1
        return {"bytes": sides * (2 * rows * d * e + 8 * b * case["tokens"]),
                "flops": sides * 3 * rows * case["rotary_dim"]}
    f = BYTES[case["format"]]
    row = d * f + (4 if case["format"] in ("fp8", "int8") else 0)
    if case["op"] == "cache":
        wrote = b * case["new"] * case["heads"]
        read = wrote if case["read"] == "new" else b * (case["context"] + case["new"]) * case["heads"]
        tokens = (wrote + read) // case["heads"]
        return {"bytes": 2 * (wrote + read) * (d * e + row) + 8 * tokens,
                "flops": 2 * (wrote + read) * d}
    keys = sum(min(n, case["window"] or n) for n in _lengths(case))
    q = b * case["q_heads"]
    return {"bytes": 2 * keys * case["heads"] * row + q * (2 * d * e + 4) + 4 * keys // case["page"],
            "flops": 4 * keys * case["q_heads"] * d}


# ---------------------------------------------------------------- 64 bits

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rotary":
        frequencies, factor = _frequencies(case)
        angle = (state["positions"].double()[..., None] * frequencies)[:, :, None]
        turn = torch.polar(torch.full_like(angle, factor), angle)  # factor * e^(i angle)
        r = case["rotary_dim"]

        def turned(x, by):
            x = x.double()
            if case["layout"] == "half":
                z = torch.complex(x[..., :r // 2].contiguous(), x[..., r // 2:r].contiguous()) * by
                head = torch.cat([z.real, z.imag], -1)
            else:
                z = torch.view_as_complex(x[..., :r].reshape(*x.shape[:-1], r // 2, 2).contiguous())
                head = torch.view_as_real(z * by).flatten(-2)
            return torch.cat([head, x[..., r:]], -1)

        out = turned(state["q"], turn), turned(state["k"], turn)
        if case["direction"] == "forward":
            return out
        return *out, turned(state["gq"], turn.conj()), turned(state["gk"], turn.conj())
    if case["op"] == "cache":
        page, form = case["page"], case["format"]
        kept = state["written"] >= 0
        slots = state["written"][kept]
        whole, scales, rows = [], [], []
        for x, data, scale in ((state["k_new"], state["k"], state["k_scale"]),
                               (state["v_new"], state["v"], state["v_scale"])):
            # the cache as one list of slots, [slot, head, channel]
            values = (data.view(torch.int8).transpose(1, 2).flatten(0, 1).view(data.dtype)
                      if form in ("fp8", "int8") else data.transpose(1, 2).flatten(0, 1)).double()
            new = x[kept].double()
            if scale is None:
                values[slots] = new
            else:
                lines = scale.transpose(1, 2).flatten(0, 1).double()
                top = new.abs().amax(-1)
                if form == "fp8":
                    step = torch.exp2(torch.ceil(torch.log2(top / 448.0)))
                    step = torch.where(top > 448.0 * step, step * 2.0, step)
                    y = new / step[..., None]
                    # the spacing of a value with 3 mantissa bits, 2^-9 below 2^-6
                    ulp = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3.0)
                    codes = torch.round(y / ulp) * ulp
                else:
                    # the scale and its reciprocal are 32-bit numbers
                    step = (top * (1.0 / torch.tensor(127.0)).double()).float().double()
                    ratio = (1.0 / step).float().double()
                    # the product is rounded to 32 bits, then to a whole number
                    codes = torch.round((new * ratio[..., None]).float().double())
                values *= lines[..., None]
                values[slots], lines[slots] = codes * step[..., None], step
                scales.append(lines.view(data.shape[0], page, -1).transpose(1, 2))
            whole.append(values)
            back = values[state["read"].clamp(min=0)]
            back[state["read"] < 0] = 0.0
            rows.append(back)
        if form in DTYPES:
            scales = [w.view(-1, page, case["heads"], case["head_dim"]).transpose(1, 2)
                      for w in whole]
        return rows[0], rows[1], scales[0], scales[1]
    heads, d = case["heads"], case["head_dim"]
    q = state["q"].double().unflatten(1, (heads, -1))
    out, lse = torch.zeros_like(q), torch.full_like(q[..., 0], float("-inf"))
    pages = state["table"].long()
    for b, n in enumerate(state["known_lengths"]):
        first = max(0, n - case["window"]) if case["window"] else 0
        held = pages[b, :-(-n // case["page"])]  # whole pages, then the keys of the window
        for h in range(heads if n else 0):
            rows = []
            for data, scale in ((state["k"], state["k_scale"]), (state["v"], state["v_scale"])):
                x = data.view(torch.int8)[:, h] if data.element_size() == 1 else data[:, h]
                x = x[held].view(data.dtype).double()
                if scale is not None:
                    x = x * scale[held, h].double().unsqueeze(-1)
                rows.append(x.view(-1, d)[first:n])
            logits = state["scale"] * (q[b, h] @ rows[0].T.contiguous())
            lse[b, h] = torch.logsumexp(logits, -1)
            out[b, h] = torch.softmax(logits, -1) @ rows[1]
    return out.flatten(1, 2), lse.flatten(1, 2)
