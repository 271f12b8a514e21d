"""The serving operators (rotary positions, cache pages, attention over packed prompts, attention of drafted tokens over
the cache) as cases that can be measured: inputs, plain forms in elementary torch operations, definitions in 64 bits."""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _ints(text):
    return [int(x) for x in text.split(",")]


def _text(values):
    return ",".join(str(v) for v in values)


# ---------------------------------------------------------------- cases
def listed():
    return [
        # one decoding step of 64 sequences: rotate Q and K, write K and V to the cache; latency counts
        dict(name="rotary append step", op="rotary", tokens=64, heads=32, kv_heads=8, dim=128, rotary=128, interleaved=False,
             scaling="none", far=8192, page=64, inverse=False, dtype="bf16"),
        # a batch of prompts of a long-context model, written to the cache
        dict(name="rotary append prompts", op="rotary", tokens=16384, heads=32, kv_heads=8, dim=128, rotary=128, interleaved=False,
             scaling="by_parts", far=1000000, page=16, inverse=False, dtype="bf16"),
        # gradients through rotary positions on half of an interleaved head, an odd token count, no cache
        dict(name="rotary gradients", op="rotary", tokens=5001, heads=16, kv_heads=4, dim=128, rotary=64, interleaved=True,
             scaling="linear", far=32768, page=0, inverse=True, dtype="fp16"),
        # after verification: the accepted path of every drafted tree moves to the front, in all layers
        dict(name="accept drafted", op="accept", layers=16, contexts=_text(500 + 37 * i for i in range(64)), drafted=32, accepted=6,
             page=64, kv_heads=8, dim=128, dtype="bf16"),
        # copy on write and defragmentation: whole pages, in all layers
        dict(name="copy pages", op="copy", layers=8, copies=256, page=64, kv_heads=8, dim=128, dtype="bf16"),
        # one short prompt: latency counts
        dict(name="prompt short", op="prompt", lengths="200", heads=32, kv_heads=8, dim=128, causal=True, dtype="bf16"),
        # a mix of prompts of different lengths, one token to some thousand, smaller heads
        dict(name="prompts ragged", op="prompt", lengths="1,777,64,2049,130,1500,333,45,1023,128,600", heads=16, kv_heads=4, dim=64,
             causal=True, dtype="fp16"),
        # full prompts at the size the framework's protected attention is quoted at
        dict(name="prompts full", op="prompt", lengths="4096,4096,4096,4096", heads=32, kv_heads=8, dim=128, causal=True, dtype="bf16"),
        # one sequence, one new token
        dict(name="decode one", op="tree", contexts="1500", drafted="1", heads=32, kv_heads=8, dim=128, page=16, dtype="bf16"),
        # a serving batch, one new token each, contexts of every length
        dict(name="decode batch", op="tree", contexts=_text(int(16 * 1.1038 ** i) for i in range(64)), drafted=_text([1] * 64), heads=32,
             kv_heads=8, dim=128, page=64, dtype="bf16"),
        # trees of drafted tokens of several sizes
        dict(name="trees batch", op="tree", contexts=_text(300 + 491 * i for i in range(16)), drafted=_text(8 + (7 * i) % 41 for i in range(16)),
             heads=32, kv_heads=8, dim=128, page=32, dtype="fp16"),
        # trees over very long contexts
        dict(name="trees long", op="tree", contexts="131072,65001", drafted="64,31", heads=32, kv_heads=8, dim=128, page=128, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "rotary", "accept", "copy", "prompt", "prompt", "prompt", "tree", "tree", "tree"])
    dtype = rng.choice(["bf16", "fp16"])
    kv_heads = rng.choice([1, 2, 4, 8])
    dim = rng.choice([64, 128])
    if op == "rotary":
        rotary = rng.choice([dim, dim, dim // 2, dim // 4])
        inverse = rng.random() < 0.3
        return dict(op=op, tokens=_log_int(rng, 1, 16384), heads=kv_heads * rng.choice([1, 2, 3, 4]), kv_heads=kv_heads, dim=dim, rotary=rotary,
                    interleaved=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "base", "by_parts"]), far=_log_int(rng, 100, 1000000),
                    page=0 if inverse else rng.choice([0, 16, 32, 64, 128]), inverse=inverse, dtype=dtype)
    if op == "accept":
        drafted = _log_int(rng, 4, 64)
        return dict(op=op, layers=rng.randint(1, 16), contexts=_text(_log_int(rng, 1, 3000) for _ in range(_log_int(rng, 1, 64))), drafted=drafted,
                    accepted=rng.randint(1, max(1, drafted // 3)), page=rng.choice([16, 32, 64, 128]), kv_heads=kv_heads, dim=dim, dtype=dtype)
    if op == "copy":
        return dict(op=op, layers=rng.randint(1, 8), copies=_log_int(rng, 1, 256), page=rng.choice([16, 32, 64]), kv_heads=kv_heads, dim=dim,
                    dtype=dtype)
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8] if kv_heads <= 4 else [1, 2, 3, 4])
    if op == "prompt":
        longest = _log_int(rng, 16, 4096)
        count = _log_int(rng, 1, max(1, min(24, 16384 // longest)))
        lengths = [longest] + [_log_int(rng, 1, longest) for _ in range(count - 1)]
        rng.shuffle(lengths)
        return dict(op=op, lengths=_text(lengths), heads=heads, kv_heads=kv_heads, dim=dim, causal=rng.random() < 0.8, dtype=dtype)
    count = _log_int(rng, 1, 64)
    most = max(200, min(131072, 200000 // count))
    one = rng.random() < 0.4
    widest = max(2, min(64, 400 // count))
    return dict(op="tree", contexts=_text(_log_int(rng, 1, most) for _ in range(count)),
                drafted=_text(1 if one else _log_int(rng, 1, widest) for _ in range(count)), heads=heads, kv_heads=kv_heads, dim=dim,
                page=rng.choice([16, 32, 64, 128]), dtype=dtype)


# ---------------------------------------------------------------- inputs
def _normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _offsets(lengths):
    return torch.tensor([0] + list(np.cumsum(lengths)), dtype=torch.int32, device="cuda")


def _frequency_options(case):
    # the scalings of long contexts at their usual settings: eight times an original context of 8192
    return {"none": dict(base=10000.0), "linear": dict(base=10000.0, scaling="linear", factor=8.0),
            "base": dict(base=10000.0, scaling="base", factor=8.0),
            "by_parts": dict(base=500000.0, scaling="by_parts", factor=8.0, original_length=8192, low=1.0, high=4.0, magnitude=1.2)}[case["scaling"]]


def _paged(rng, lengths, page):
    """A page table for sequences of these lengths, pages in random order, a few pages spare; entries behind the last page: -1."""
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + 3
    order = rng.permutation(pages)
    table = np.full((len(lengths), max(need)), -1, dtype=np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return pages, table


def _tree_words(rng, drafted):
    """Visibility of every drafted token, packed: bit j of row i is set where j is i or one of its ancestors."""
    words = max(1, -(-max(drafted) // 32))
    rows = np.zeros((sum(drafted), words), dtype=np.uint32)
    at = 0
    for n in drafted:
        seen = np.zeros((n, words), dtype=np.uint32)
        for i in range(n):
            if i:
                seen[i] = seen[rng.randint(max(0, i - 8), i)]
            seen[i, i >> 5] |= np.uint32(1 << (i & 31))
        rows[at:at + n] = seen
        at += n
    return torch.from_numpy(rows.view(np.int32)).cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.RandomState(seed & 0x7FFFFFFF)
    dtype = DTYPES[case["dtype"]]
    kv_heads, dim = case["kv_heads"], case["dim"]
    s = {"case": case}
    if case["op"] == "rotary":
        tokens = case["tokens"]
        s["q"] = _normal(gen, (tokens, case["heads"], dim), dtype)
        s["k"] = _normal(gen, (tokens, kv_heads, dim), dtype)
        s["positions"] = torch.randint(0, case["far"], (tokens,), generator=gen, device="cuda")
        s["q_out"] = torch.empty_like(s["q"])
        if case["page"]:
            page = case["page"]
            pages = -(-tokens // page) + 2
            s["v"] = _normal(gen, (tokens, kv_heads, dim), dtype)
            s["k_cache"] = _normal(gen, (1, pages, page, kv_heads, dim), dtype)
            s["v_cache"] = _normal(gen, (1, pages, page, kv_heads, dim), dtype)
            if tokens <= 256:  # one token of every sequence: anywhere
                slots = rng.permutation(pages * page)[:tokens]
            else:  # whole prompts: page by page
                slots = (rng.permutation(pages)[:, None] * page + np.arange(page)).reshape(-1)[:tokens]
            s["slots"] = torch.from_numpy(slots.astype(np.int64)).cuda()
        else:
            s["k_out"] = torch.empty_like(s["k"])
        if own:
            import ft_gemm_b200 as ftg
            s["rotary"] = ftg.Rotary(dim, rotary_dim=case["rotary"], interleaved=case["interleaved"], **_frequency_options(case))
            if case["page"]:
                s["cache"] = ftg.PagedCache(s["k_cache"], s["v_cache"])
    elif case["op"] == "copy":
        copies = case["copies"]
        shape = (case["layers"], 2 * copies + 5, case["page"], kv_heads, dim)
        s["k_cache"], s["v_cache"] = _normal(gen, shape, dtype), _normal(gen, shape, dtype)
        order = rng.permutation(2 * copies + 5).astype(np.int32)
        s["sources"], s["targets"] = (torch.from_numpy(order[i * copies:(i + 1) * copies].copy()).cuda() for i in (0, 1))
        if own:
            import ft_gemm_b200 as ftg
            s["cache"] = ftg.PagedCache(s["k_cache"], s["v_cache"])
    elif case["op"] == "accept":
        contexts, n, most = _ints(case["contexts"]), case["drafted"], case["accepted"]
        pages, table = _paged(rng, [c + n for c in contexts], case["page"])
        shape = (case["layers"], pages, case["page"], kv_heads, dim)
        s["k_cache"], s["v_cache"] = _normal(gen, shape, dtype), _normal(gen, shape, dtype)
        s["table"] = torch.from_numpy(table).cuda()
        s["lengths"] = torch.tensor([c + n for c in contexts], dtype=torch.int32, device="cuda")
        s["drafted"] = _offsets([n] * len(contexts))
        paths, counts = [], []
        for _ in contexts:
            # a path from the root: some first children, then nodes further back than the path is long
            count = rng.randint(1, most + 1)
            same = rng.randint(1, count + 1)
            paths += list(range(same)) + sorted(int(x) for x in count + rng.permutation(n - count)[:count - same])
            counts.append(count)
        s["accepted"] = torch.tensor(paths, dtype=torch.int32, device="cuda")
        s["accepted_offsets"] = _offsets(counts)
        s["new_lengths"] = torch.empty_like(s["lengths"])
        if own:
            import ft_gemm_b200 as ftg
            s["cache"] = ftg.PagedCache(s["k_cache"], s["v_cache"])
    elif case["op"] == "prompt":
        lengths = _ints(case["lengths"])
        s["q"] = _normal(gen, (sum(lengths), case["heads"], dim), dtype, 1.5)
        s["k"] = _normal(gen, (sum(lengths), kv_heads, dim), dtype)
        s["v"] = _normal(gen, (sum(lengths), kv_heads, dim), dtype)
        s["offsets"] = _offsets(lengths)
        s["out"] = torch.empty_like(s["q"])
        if own:
            import ft_gemm_b200 as ftg
            s["attention"] = ftg.PromptAttention(case["heads"], kv_heads, dim, dtype=dtype, causal=case["causal"])
    else:
        contexts, drafted = _ints(case["contexts"]), _ints(case["drafted"])
        lengths = [c + n for c, n in zip(contexts, drafted)]
        pages, table = _paged(rng, lengths, case["page"])
        s["q"] = _normal(gen, (sum(drafted), case["heads"], dim), dtype, 1.5)
        shape = (1, pages, case["page"], kv_heads, dim)
        s["k_cache"], s["v_cache"] = _normal(gen, shape, dtype), _normal(gen, shape, dtype)
        s["table"] = torch.from_numpy(table).cuda()
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        s["offsets"] = _offsets(drafted)
        s["mask"] = _tree_words(rng, drafted)
        s["out"] = torch.empty_like(s["q"])
        if own:
            import ft_gemm_b200 as ftg
            s["cache"] = ftg.PagedCache(s["k_cache"], s["v_cache"])
            s["attention"] = ftg.TreeAttention(case["heads"], s["cache"])
    return s


# ---------------------------------------------------------------- plain forms
def _plain_frequencies(case, device):
    o = _frequency_options(case)
    r = case["rotary"]
    base = o["base"] * o["factor"] ** (r / (r - 2)) if case["scaling"] == "base" else o["base"]
    f = base ** (-torch.arange(0, r, 2, dtype=torch.float64, device=device) / r)
    if case["scaling"] == "linear":
        f = f / o["factor"]
    if case["scaling"] == "by_parts":
        keep = ((o["original_length"] * f / (2 * math.pi) - o["low"]) / (o["high"] - o["low"])).clamp(0, 1)
        f = f * (keep + (1 - keep) / o["factor"])
    return f, o.get("magnitude", 1.0)


def _plain_rotate(x, cos, sin, rotary, interleaved):
    x = x.float()
    y = x.clone()
    a, b = (x[..., 0:rotary:2], x[..., 1:rotary:2]) if interleaved else (x[..., :rotary // 2], x[..., rotary // 2:rotary])
    c, d = (y[..., 0:rotary:2], y[..., 1:rotary:2]) if interleaved else (y[..., :rotary // 2], y[..., rotary // 2:rotary])
    c.copy_(a * cos - b * sin)
    d.copy_(a * sin + b * cos)
    return y


def _plain_softmax_product(scores, visible, v):
    """softmax over the visible keys times v; rows that see nothing give zeros."""
    scores = scores.masked_fill(~visible, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)


def _plain_padded(lengths, device):
    """Row of every (sequence, place) in the packed order, and whether there is one."""
    start = torch.cumsum(lengths, 0) - lengths
    place = torch.arange(int(lengths.max()), device=device)
    there = place[None] < lengths[:, None]
    return torch.where(there, start[:, None] + place[None], torch.zeros_like(start[:, None])), there


def _plain(s):
    case = s["case"]
    dim, kv_heads = case["dim"], case["kv_heads"]
    if case["op"] == "rotary":
        f, magnitude = _plain_frequencies(case, s["q"].device)
        angle = s["positions"].double()[:, None] * f
        cos, sin = ((magnitude * g(angle)).float()[:, None, :] for g in (torch.cos, torch.sin))
        sin = -sin if case["inverse"] else sin
        s["q_out"].copy_(_plain_rotate(s["q"], cos, sin, case["rotary"], case["interleaved"]))
        k = _plain_rotate(s["k"], cos, sin, case["rotary"], case["interleaved"])
        if not case["page"]:
            s["k_out"].copy_(k)
            return [s["q_out"], s["k_out"]]
        s["k_cache"].view(-1, kv_heads, dim)[s["slots"]] = k.to(s["k"].dtype)
        s["v_cache"].view(-1, kv_heads, dim)[s["slots"]] = s["v"]
        return [s["q_out"], s["k_cache"], s["v_cache"]]
    if case["op"] == "copy":
        source, target = s["sources"].long(), s["targets"].long()
        s["k_cache"][:, target] = s["k_cache"][:, source]
        s["v_cache"][:, target] = s["v_cache"][:, source]
        return [s["k_cache"], s["v_cache"]]
    if case["op"] == "accept":
        page, layers = case["page"], case["layers"]
        counts = (s["accepted_offsets"][1:] - s["accepted_offsets"][:-1]).long()
        base = (s["lengths"] - (s["drafted"][1:] - s["drafted"][:-1])).long()
        which = torch.repeat_interleave(torch.arange(len(base), device=base.device), counts, output_size=len(s["accepted"]))
        place = torch.arange(len(which), device=base.device) - s["accepted_offsets"][:-1].long()[which]
        old, new = base[which] + s["accepted"].long(), base[which] + place
        old, new = (s["table"].long()[which, x // page] * page + x % page for x in (old, new))
        for cache in (s["k_cache"].view(layers, -1, kv_heads, dim), s["v_cache"].view(layers, -1, kv_heads, dim)):
            cache[:, new] = cache[:, old]
        s["new_lengths"].copy_(base + counts)
        return [s["k_cache"], s["v_cache"], s["new_lengths"]]
    group = case["heads"] // kv_heads
    lengths = (s["offsets"][1:] - s["offsets"][:-1]).long()
    rows, there = _plain_padded(lengths, s["q"].device)
    q = s["q"].float()[rows]  # [sequence, query, head, dim]
    batch, most = rows.shape
    q = q.view(batch, most, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, group * most, dim)
    if case["op"] == "prompt":
        k, v = (torch.where(there[..., None, None], s[x].float()[rows], 0.0).permute(0, 2, 1, 3) for x in "kv")
        visible = there[:, None, :].expand(batch, most, most)
        if case["causal"]:
            visible = visible & torch.ones(most, most, dtype=torch.bool, device=rows.device).tril()
    else:
        total = s["lengths"].long()
        key = torch.arange(int(total.max()), device=rows.device)
        stored = key[None] < total[:, None]
        slot = torch.where(stored, s["table"].long()[:, key // case["page"]] * case["page"] + key % case["page"], 0)
        k, v = (torch.where(stored[..., None, None], s[x].view(-1, kv_heads, dim)[slot].float(), 0.0).permute(0, 2, 1, 3) for x in ("k_cache", "v_cache"))
        node = key[None] - (total - lengths)[:, None]  # [sequence, key]: which drafted token a key is, negative before them
        words = s["mask"].long()[rows]  # [sequence, query, word]
        word = (node // 32).clamp(0, words.shape[-1] - 1)[:, None, :].expand(batch, most, len(key))
        bit = (torch.gather(words, 2, word) >> (node % 32)[:, None, :]) & 1
        visible = stored[:, None, :] & ((node < 0)[:, None, :] | (bit == 1))
    scores = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(dim)
    seen = visible[:, None, None].expand(batch, 1, group, most, visible.shape[-1]).reshape(batch, 1, group * most, visible.shape[-1])
    o = _plain_softmax_product(scores, seen, v)
    o = o.view(batch, kv_heads, group, most, dim).permute(0, 3, 1, 2, 4).reshape(batch, most, case["heads"], dim)
    s["out"].copy_(o[there])
    return [s["out"]]


def run(s):
    if not own:
        return _plain(s)
    case = s["case"]
    if case["op"] == "rotary":
        if case["page"]:
            s["cache"].append(0, s["k"], s["v"], s["slots"], rotary=s["rotary"], positions=s["positions"], q=s["q"], q_out=s["q_out"])
            return [s["q_out"], s["k_cache"], s["v_cache"]]
        s["rotary"].run(s["q"], s["k"], s["positions"], s["q_out"], s["k_out"], inverse=case["inverse"])
        return [s["q_out"], s["k_out"]]
    if case["op"] == "copy":
        s["cache"].copy_pages(s["sources"], s["targets"])
        return [s["k_cache"], s["v_cache"]]
    if case["op"] == "accept":
        s["cache"].accept(s["table"], s["lengths"], s["drafted"], s["accepted"], s["accepted_offsets"], s["new_lengths"])
        return [s["k_cache"], s["v_cache"], s["new_lengths"]]
    if case["op"] == "prompt":
        s["attention"].run(s["q"], s["k"], s["v"], s["out"], s["offsets"])
    else:
        s["attention"].run(s["q"], 0, s["offsets"], s["table"], s["lengths"], s["out"], mask=s["mask"])
    return [s["out"]]


# ---------------------------------------------------------------- what cannot be done without
def work(case):
    kv_heads, dim = case["kv_heads"], case["dim"]
    kv_row = kv_heads * dim * 2
    if case["op"] == "rotary":
        q_row = case["heads"] * dim * 2
        token = 2 * q_row + 2 * kv_row + 8 + (2 * kv_row + 8 if case["page"] else 0)
        return {"bytes": case["tokens"] * token, "flops": case["tokens"] * (case["heads"] + kv_heads) * case["rotary"] * 3}
    if case["op"] == "copy":
        return {"bytes": case["layers"] * case["copies"] * case["page"] * kv_row * 4 + 8 * case["copies"], "flops": 0}
    if case["op"] == "accept":
        # between one token and `accepted` move in each sequence
        moved = len(_ints(case["contexts"])) * (case["accepted"] + 1) / 2
        return {"bytes": case["layers"] * moved * kv_row * 4 + 4 * moved + 16 * len(_ints(case["contexts"])), "flops": 0}
    if case["op"] == "prompt":
        lengths = _ints(case["lengths"])
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lengths)
        queries, keys = sum(lengths), sum(lengths)
    else:
        contexts, drafted = _ints(case["contexts"]), _ints(case["drafted"])
        pairs = sum(n * c + n * (n + 1) // 2 for c, n in zip(contexts, drafted))
        queries, keys = sum(drafted), sum(contexts) + sum(drafted)
    return {"bytes": 4 * queries * case["heads"] * dim + 2 * keys * kv_row, "flops": 4 * pairs * case["heads"] * dim}


# ---------------------------------------------------------------- definitions in 64 bits
def _exact_rotary(case, s):
    o, r = _frequency_options(case), case["rotary"]
    f = []
    for i in range(r // 2):
        base = o["base"]
        if case["scaling"] == "base":
            base = base * 8.0 ** (r / (r - 2))
        w = math.exp(-2.0 * i / r * math.log(base))
        if case["scaling"] == "linear":
            w = w / 8.0
        if case["scaling"] == "by_parts":
            turns = 8192 * w / (2 * math.pi)
            g = min(1.0, max(0.0, (turns - 1.0) / 3.0))
            w = (1.0 - g) * w / 8.0 + g * w
        f.append(w)
    theta = torch.outer(s["positions"].double(), torch.tensor(f, dtype=torch.float64, device="cuda"))
    turn = torch.polar(torch.full_like(theta, o.get("magnitude", 1.0)), -theta if case["inverse"] else theta)[:, None]

    def rotate(x):
        x = x.double()
        head = x[..., :r]
        z = torch.view_as_complex(head.reshape(*head.shape[:-1], r // 2, 2).contiguous()) if case["interleaved"] else torch.complex(head[..., :r // 2], head[..., r // 2:])
        z = z * turn
        head = torch.view_as_real(z).flatten(-2) if case["interleaved"] else torch.cat([z.real, z.imag], -1)
        return torch.cat([head, x[..., r:]], -1)

    if not case["page"]:
        return [rotate(s["q"]), rotate(s["k"])]
    k, v = s["k_cache"].double(), s["v_cache"].double()
    k.flatten(0, 2)[s["slots"]] = rotate(s["k"])
    v.flatten(0, 2)[s["slots"]] = s["v"].double()
    return [rotate(s["q"]), k, v]


def _exact_head(q, k, v, visible):
    """One sequence and one key head: q [group, n, dim], k, v [m, dim], visible [n, m] or None."""
    x = torch.einsum("gnd,md->gnm", q, k) * q.shape[-1] ** -0.5
    if visible is not None:
        x = torch.where(visible, x, torch.full_like(x, -math.inf))
    return torch.einsum("gnm,md->gnd", torch.nan_to_num(torch.softmax(x, -1)), v)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(case, s)
    if case["op"] == "copy":
        for name in ("k_cache", "v_cache"):
            for a, b in zip(s["sources"].tolist(), s["targets"].tolist()):
                s[name][:, b].copy_(s[name][:, a])
        return [s["k_cache"].double(), s["v_cache"].double()]
    if case["op"] == "accept":
        page, at, ends = case["page"], s["accepted"].tolist(), s["accepted_offsets"].tolist()
        table, lengths = s["table"].tolist(), []
        for b, context in enumerate(_ints(case["contexts"])):
            for i, node in enumerate(at[ends[b]:ends[b + 1]]):
                old, new = context + node, context + i
                for name in ("k_cache", "v_cache"):
                    s[name][:, table[b][new // page], new % page] = s[name][:, table[b][old // page], old % page]
            lengths.append(context + ends[b + 1] - ends[b])
        return [s["k_cache"].double(), s["v_cache"].double(), torch.tensor(lengths, dtype=torch.int32)]
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    starts = s["offsets"].tolist()
    for b in range(len(starts) - 1):
        lo, hi = starts[b], starts[b + 1]
        n = hi - lo
        if case["op"] == "prompt":
            keys, values = s["k"][lo:hi], s["v"][lo:hi]
            visible = torch.arange(n, device="cuda")[None] <= torch.arange(n, device="cuda")[:, None] if case["causal"] else None
        else:
            m = int(s["lengths"][b])
            pages = s["table"][b, :-(-m // case["page"])].long()
            keys, values = (s[x][0][pages].flatten(0, 1)[:m] for x in ("k_cache", "v_cache"))
            bits = np.unpackbits(s["mask"][lo:hi].cpu().numpy().view(np.uint8), axis=1, bitorder="little")[:, :n]
            visible = torch.ones(n, m, dtype=torch.bool, device="cuda")
            visible[:, m - n:] = torch.from_numpy(bits.astype(bool)).cuda()
        for h in range(case["kv_heads"]):
            q = s["q"][lo:hi, h * group:(h + 1) * group].double().transpose(0, 1)
            out[lo:hi, h * group:(h + 1) * group] = _exact_head(q, keys[:, h].double(), values[:, h].double(), visible).transpose(0, 1)
    return [out]
