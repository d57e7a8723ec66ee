"""Cases of the serving step of an attention layer over a paged key/value cache:
the rotary embedding with positions of several axes, the write of new keys and
values into pages (as they are or in 8 bits), the read back into dense tiles and
the attention of a few new tokens over the pages.

Layouts: pages [n_pages, n_head_kv, page_rows, head]; table [n_batch, max_pages]
and lens [n_batch] int32 (lens counts the newest rows); tiles [entries, rows, head]
with entry = sequence + n_batch * head index; 8-bit pages are e4m3 with one power of
two per row, held as its exponent + 127.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
LARGEST = 4.2e8         # bytes of the largest listed case


def _rope(name, dtype, n_batch, seq, heads_q, heads_k, head, n_axes, backward, far=0):
    return {"name": name, "op": "rope", "dtype": dtype, "n_batch": n_batch, "seq": seq,
            "heads_q": heads_q, "heads_k": heads_k, "head": head, "n_axes": n_axes,
            "backward": backward, "far": far}


def _paged(name, op, dtype, packed, n_batch, heads_kv, head, page_rows, longest, shortest,
           rows=1, kv_group=1, padded=False):
    """longest, shortest: the lengths of the sequences run between the two, spread over
    their logarithm.  rows: new tokens a sequence (append, attend), rows read (read).
    padded: some sequences bring fewer tokens than that."""
    return {"name": name, "op": op, "dtype": dtype, "packed": packed, "n_batch": n_batch,
            "heads_kv": heads_kv, "head": head, "page_rows": page_rows, "longest": longest,
            "shortest": shortest, "rows": rows, "kv_group": kv_group, "padded": padded}


def listed():
    return [
        # a generation step of eight sequences: one token each, 32 query and 8 key heads
        _rope("rope_token", "bf16", 8, 1, 32, 8, 128, 1, False, far=5000),
        # four images of 7 x 143 patches (rows and columns), a small fp32 model of 12 heads
        _rope("rope_image_fp32", "fp32", 4, 1001, 12, 12, 64, 2, False),
        # the gradient over a prompt of 4096 video patches (time, height, width)
        _rope("rope_video_backward", "bf16", 1, 4096, 32, 8, 128, 3, True),
        # a generation step: one row a sequence and head, written in 8 bits
        _paged("append_token_8bit", "append", "bf16", True, 8, 8, 128, 64, 8192, 500),
        # prompts of up to 4096 tokens of a padded batch, written in 8 bits
        _paged("append_prompt_8bit", "append", "fp16", True, 4, 8, 128, 32, 5000, 4096, rows=4096,
               padded=True),
        # a short odd piece of an unpacked fp32 cache, for a chunk that goes on with it
        _paged("read_chunk_fp32", "read", "fp32", False, 3, 12, 64, 16, 1038, 700, rows=1001),
        # the whole of eight caches of 8192 tokens back in 16 bits
        _paged("read_whole_8bit", "read", "bf16", True, 8, 8, 128, 64, 8192, 8192, rows=8192),
        # one user's generation step at a short context: latency
        _paged("attend_one_user", "attend", "bf16", False, 1, 8, 128, 64, 1001, 1001, kv_group=4),
        # a small fp32 model, four sequences of 1024 tokens, no sharing of heads
        _paged("attend_small_fp32", "attend", "fp32", False, 4, 12, 64, 32, 1024, 1024),
        # the decode workload: 16 new tokens over 8192, 32 query heads on 8
        _paged("attend_decode", "attend", "bf16", False, 8, 8, 128, 128, 8192, 8192, rows=16,
               kv_group=4),
        # serving: 64 sequences of 17 to 16384 tokens, 8-bit pages of 16 rows
        _paged("attend_ragged_8bit", "attend", "bf16", True, 64, 8, 128, 16, 16384, 17,
               kv_group=4),
        # four drafted tokens to check, fewer in some of the sequences, 8 query heads on one
        _paged("attend_drafts_8bit", "attend", "fp16", True, 16, 8, 64, 64, 4096, 300, rows=4,
               kv_group=8, padded=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["rope", "append", "read", "attend", "attend"])
        head = rng.choice([64, 128])
        n_batch = _log(rng, 1, 64)
        heads_kv = rng.choice([1, 2, 4, 8, 12, 16])
        kv_group = rng.choice([1, 1, 2, 4, 8])
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        if op == "rope":
            n_axes = rng.choice([1, 2, 3])
            c = _rope("", dtype, n_batch, _log(rng, 1, 8192), heads_kv * kv_group, heads_kv, head,
                      n_axes, rng.random() < 0.5, far=rng.choice([0, 0, 100000]))
        else:
            packed = dtype != "fp32" and rng.random() < 0.5
            longest = _log(rng, 1, 16384)
            shortest = longest if rng.random() < 0.4 else _log(rng, 1, longest)
            most = {"append": shortest, "read": longest, "attend": min(16, shortest)}[op]
            rows = 1 if rng.random() < 0.3 else _log(rng, 1, most)
            c = _paged("", op, dtype, packed, n_batch, heads_kv, head,
                       rng.choice([16, 32, 64, 128, 256]), longest, shortest, rows=rows,
                       kv_group=kv_group if op == "attend" else 1,
                       padded=op != "read" and rng.random() < 0.3)
        if work(c)["bytes"] <= LARGEST and _plain_bytes(c) <= 1.5e10 and _pool_bytes(c) <= 2e9:
            del c["name"]
            return c


def _lens(case):
    """The sequences' lengths in ascending order; prepare() shuffles them."""
    n, lo, hi = case["n_batch"], case["shortest"], case["longest"]
    return [hi if n == 1 else int(round(math.exp(math.log(lo) + (math.log(hi) - math.log(lo)) * i / (n - 1))))
            for i in range(n)]


def _new_rows(case):
    """How many of the `rows` new tokens each sequence brings, in the order of _lens."""
    n, rows = case["n_batch"], case["rows"]
    if not case["padded"]:
        return [rows] * n
    return [rows - (rows * (i % 4)) // 4 for i in range(n)]


def _pool_bytes(case):
    if case["op"] == "rope":
        return 0
    pages = sum(-(-l // case["page_rows"]) for l in _lens(case))
    e = 1 if case["packed"] else BYTES[case["dtype"]]
    return 2.0 * pages * case["page_rows"] * case["heads_kv"] * case["head"] * e


def _plain_bytes(case):
    """What the plain form holds at most: padded fp32 copies of keys and values."""
    if case["op"] != "attend":
        return 0
    return 8.0 * case["n_batch"] * case["heads_kv"] * case["longest"] * (case["head"] + case["rows"] * case["kv_group"])


def work(case):
    e = BYTES[case["dtype"]]
    head = case["head"]
    if case["op"] == "rope":
        tokens = case["n_batch"] * case["seq"]
        values = tokens * (case["heads_q"] + case["heads_k"]) * head
        return {"bytes": 2 * e * values + 8 * tokens * case["n_axes"], "flops": 3 * values}
    stored = head + 1 if case["packed"] else head * e       # bytes of a row in its page
    if case["op"] == "attend":
        rows, group = case["rows"], case["kv_group"]
        lens = _lens(case)
        entries = case["n_batch"] * case["heads_kv"] * group
        bytes_ = 2 * sum(lens) * case["heads_kv"] * stored + 2 * entries * rows * head * e + 4 * entries * rows
        pairs = sum(new * l - new * (new - 1) // 2 for l, new in zip(lens, _new_rows(case)))
        return {"bytes": bytes_, "flops": 4 * pairs * head * case["heads_kv"] * group}
    if case["op"] == "append":
        moved = sum(_new_rows(case)) * case["heads_kv"]
        return {"bytes": 2 * moved * (head * e + stored), "flops": 4 * moved * head}
    first = case["longest"] - case["rows"]
    there = sum(max(0, l - first) for l in _lens(case)) * case["heads_kv"]
    out = case["n_batch"] * case["heads_kv"] * case["rows"]
    return {"bytes": 2 * (there * stored + out * head * e), "flops": 2 * there * head}


def _sections(head, n_axes):
    """Pairs of each axis: even shares, what is left over to the first."""
    share = (head // 2) // n_axes
    return [head // 2 - share * (n_axes - 1)] + [share] * (n_axes - 1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = TYPES[case["dtype"]]
    head, n_batch = case["head"], case["n_batch"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).to(dt)

    def whole(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=gen, device="cuda")

    if case["op"] == "rope":
        seq, n_axes = case["seq"], case["n_axes"]
        # time counts on from the start of the sequence, rows and columns are those of a patch
        base, step = whole(0, case["far"] + 1, n_batch, 1), torch.arange(seq, device="cuda")[None, :]
        side = max(1, int(math.sqrt(seq)))
        of_axes = {1: [step], 2: [step // side, step % side], 3: [step // side, step // side, step % side]}[n_axes]
        positions = torch.stack([base + of_axes[0]] + [x.expand(n_batch, seq) for x in of_axes[1:]])
        freqs = torch.pow(torch.tensor(10000.0, dtype=torch.float64),
                          -torch.arange(0, head, 2, dtype=torch.float64) / head).cuda()
        axes = torch.cat([torch.full((n,), a, dtype=torch.int32)
                          for a, n in enumerate(_sections(head, n_axes))]).cuda()
        q = normal(case["heads_q"] * n_batch, seq, head)
        k = normal(case["heads_k"] * n_batch, seq, head)
        return {"case": case, "positions": positions, "freqs": freqs, "axes": axes, "q": q, "k": k,
                "q_out": torch.empty_like(q), "k_out": torch.empty_like(k)}

    page_rows, heads = case["page_rows"], case["heads_kv"]
    order = torch.randperm(n_batch, generator=gen, device="cuda")
    lens = torch.tensor(_lens(case), dtype=torch.int32, device="cuda")[order]
    new_rows = torch.tensor(_new_rows(case), dtype=torch.int32, device="cuda")[order]
    max_pages = -(-case["longest"] // page_rows)
    n_pages = sum(-(-l // page_rows) for l in _lens(case))
    # a pool that has been in use for long: the pages lie in any order
    pages_of = (lens + page_rows - 1) // page_rows
    first_of = torch.cumsum(pages_of, 0) - pages_of
    at = torch.arange(max_pages, device="cuda")
    held = at[None, :] < pages_of[:, None]
    shuffled = torch.randperm(n_pages, generator=gen, device="cuda")
    table = torch.where(held, shuffled[(first_of[:, None] + at).clamp(max=n_pages - 1)], -1).to(torch.int32).contiguous()
    # (one page behind the pool: where the plain form puts the rows that nobody wants)
    shape = (n_pages + 1, heads, page_rows, head)
    if case["packed"]:
        k_pages, v_pages = ((3e2 * torch.rand(shape, generator=gen, device="cuda") - 150.0).to(torch.float8_e4m3fn)
                            for _ in range(2))
        k_scales, v_scales = (whole(117, 120, *shape[:3]).to(torch.uint8) for _ in range(2))
    else:
        k_pages, v_pages = normal(*shape), normal(*shape)
        k_scales = v_scales = None
    s = {"case": case, "k_pages": k_pages, "v_pages": v_pages, "k_scales": k_scales, "v_scales": v_scales,
         "table": table, "lens": lens, "new_rows": new_rows if case["padded"] else None, "given": new_rows}
    entries, rows = n_batch * heads, case["rows"]
    if case["op"] == "append":
        s["k"], s["v"] = normal(entries, rows, head), normal(entries, rows, head)
    elif case["op"] == "read":
        s["k"] = torch.empty(entries, rows, head, dtype=dt, device="cuda")
        s["v"] = torch.empty_like(s["k"])
    else:
        s["q"] = normal(entries * case["kv_group"], rows, head)
        s["A"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(entries * case["kv_group"], rows, dtype=torch.float32, device="cuda")
        # memory for what the shares of a long cache leave for each other, kept between steps
        s["workspace"] = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    return s


def run(s):
    return _run_own(s) if own else {"rope": _plain_rope, "append": _plain_append, "read": _plain_read,
                                    "attend": _plain_attend}[s["case"]["op"]](s)


def _run_own(s):
    from nntile_amd import hip_sdpa as h
    c = s["case"]
    if c["op"] == "rope":
        h.rope_axes(s["positions"], s["freqs"], s["axes"], s["q"], s["q_out"], s["k"], s["k_out"],
                    backward=c["backward"])
        return s["q_out"], s["k_out"]
    k_pages, v_pages = s["k_pages"][:-1], s["v_pages"][:-1]
    k_scales = v_scales = None
    if c["packed"]:
        k_scales, v_scales = s["k_scales"][:-1], s["v_scales"][:-1]
    if c["op"] == "append":
        h.paged_kv_append(s["k"], s["v"], k_pages, v_pages, s["table"], s["lens"], k_scales, v_scales,
                          new_rows=s["new_rows"])
        return k_pages, v_pages, k_scales, v_scales
    if c["op"] == "read":
        h.paged_kv_read(k_pages, v_pages, s["table"], s["lens"], s["k"], s["v"],
                        first=c["longest"] - c["rows"], k_scales=k_scales, v_scales=v_scales)
        return s["k"], s["v"]
    h.sdpa_fwd_paged(k_pages, v_pages, s["table"], s["lens"], s["q"], s["lse"], s["A"], h.MASK_CAUSAL,
                     c["kv_group"], s["workspace"], k_scales=k_scales, v_scales=v_scales,
                     new_rows=s["new_rows"], flags=h.OVERWRITE)
    return s["A"], s["lse"]


# ---- plain forms: elementary torch operations in 32 bits -------------------------

def _plain_rope(s):
    c = s["case"]
    angle = (s["positions"].to(torch.float64)[s["axes"].long()] * s["freqs"][:, None, None]).permute(1, 2, 0)
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()      # [n_batch, seq, pairs]
    if c["backward"]:
        sin = -sin

    def turned(x):
        y = x.float().reshape(-1, c["n_batch"], c["seq"], c["head"] // 2, 2)
        a, b = y[..., 0], y[..., 1]
        return torch.stack((cos * a - sin * b, sin * a + cos * b), dim=-1).reshape(x.shape).to(x.dtype)

    return turned(s["q"]), turned(s["k"])


def _rows_of(s, position, wanted):
    """The flat page rows [n_batch, heads, positions] of every head's row at `position`
    [n_batch, positions]; the spare page's where `wanted` is false."""
    c = s["case"]
    page_rows, heads = c["page_rows"], c["heads_kv"]
    page = torch.gather(s["table"].long(), 1, (position // page_rows).clamp(0, s["table"].shape[1] - 1))
    page = torch.where(wanted, page, s["k_pages"].shape[0] - 1)
    head = torch.arange(heads, device="cuda")[None, :, None]
    return (page[:, None, :] * heads + head) * page_rows + (position % page_rows)[:, None, :]


def _plain_append(s):
    c = s["case"]
    n_batch, heads, head, rows = c["n_batch"], c["heads_kv"], c["head"], c["rows"]
    r = torch.arange(rows, device="cuda")[None, :]
    new = s["given"][:, None]
    at = _rows_of(s, (s["lens"][:, None] - new + r).clamp(min=0), r < new).reshape(-1)
    for x, pages, scales in ((s["k"], s["k_pages"], s["k_scales"]), (s["v"], s["v_pages"], s["v_scales"])):
        x = x.reshape(heads, n_batch, rows, head).transpose(0, 1).reshape(-1, head)
        if c["packed"]:
            f = x.float()
            mantissa, exponent = torch.frexp(f.abs().amax(dim=-1))
            # the smallest power of two that leaves no value of the row above 448 = 0.875 * 2^9
            k = torch.where(mantissa > 0.875, exponent - 8, exponent - 9).clamp(min=-126)
            k = torch.where(mantissa == 0, -126, k)
            codes = torch.ldexp(f, -k[:, None]).to(torch.float8_e4m3fn)
            pages.view(torch.uint8).view(-1, head)[at] = codes.view(torch.uint8)
            scales.view(-1)[at] = (k + 127).to(torch.uint8)
        else:
            pages.view(-1, head)[at] = x
    if c["packed"]:
        return s["k_pages"][:-1], s["v_pages"][:-1], s["k_scales"][:-1], s["v_scales"][:-1]
    return s["k_pages"][:-1], s["v_pages"][:-1], None, None


def _plain_rows(s, pages, scales, at):
    """The page rows `at`, as fp32 values."""
    head = s["case"]["head"]
    if scales is None:
        return pages.view(-1, head)[at].float()
    codes = pages.view(torch.uint8).view(-1, head)[at].view(torch.float8_e4m3fn).float()
    return torch.ldexp(codes, scales.view(-1)[at].int()[..., None] - 127)


def _plain_read(s):
    c = s["case"]
    n_batch, heads, head, rows = c["n_batch"], c["heads_kv"], c["head"], c["rows"]
    position = torch.arange(c["longest"] - rows, c["longest"], device="cuda")[None, :].expand(n_batch, rows)
    there = position < s["lens"][:, None]
    at = _rows_of(s, position, there)
    out = []
    for pages, scales in ((s["k_pages"], s["k_scales"]), (s["v_pages"], s["v_scales"])):
        x = torch.where(there[:, None, :, None], _plain_rows(s, pages, scales, at), 0.0)
        out.append(x.transpose(0, 1).reshape(heads * n_batch, rows, head).to(TYPES[c["dtype"]]))
    return tuple(out)


def _plain_attend(s):
    c = s["case"]
    n_batch, heads, head, rows, group = c["n_batch"], c["heads_kv"], c["head"], c["rows"], c["kv_group"]
    position = torch.arange(c["longest"], device="cuda")[None, :].expand(n_batch, c["longest"])
    there = position < s["lens"][:, None]
    at = _rows_of(s, position, there)
    k = _plain_rows(s, s["k_pages"], s["k_scales"], at)                # [n_batch, heads, longest, head]
    v = torch.where(there[:, None, :, None], _plain_rows(s, s["v_pages"], s["v_scales"], at), 0.0)
    q = s["q"].float().reshape(heads, group, n_batch, rows, head).permute(2, 0, 1, 3, 4)
    q = q.reshape(n_batch, heads, group * rows, head)
    score = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(head))
    j = torch.arange(rows, device="cuda")
    last = s["lens"][:, None] - s["given"][:, None] + j                # the last key a query sees
    seen = (position[:, None, :] <= last[:, :, None]) & (j < s["given"][:, None])[:, :, None] & there[:, None, :]
    seen = seen[:, None, None].expand(n_batch, heads, group, rows, c["longest"]).reshape(score.shape)
    score = torch.where(seen, score, -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    weight = torch.exp(score - top)
    total = weight.sum(dim=-1, keepdim=True)
    A = torch.matmul(weight, v) / torch.where(total == 0, 1.0, total)
    lse = torch.log(total) + top

    def back(x):
        x = x.reshape(n_batch, heads, group, rows, x.shape[-1]).permute(1, 2, 0, 3, 4)
        return x.reshape(heads * group * n_batch, rows, x.shape[-1])

    return back(A).to(TYPES[c["dtype"]]), back(lse).squeeze(-1)


# ---- the operators' definitions in 64 bits ----------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "append": _exact_append, "read": _exact_read, "attend": _exact_attend}[case["op"]](s)


def _exact_rope(s):
    """A pair is a complex number, turned by its angle (backwards for the gradient)."""
    c = s["case"]
    out = []
    for x in (s["q"], s["k"]):
        z = torch.view_as_complex(x.double().reshape(x.shape[0], c["seq"], c["head"] // 2, 2))
        for i in range(c["head"] // 2):
            angle = s["positions"][int(s["axes"][i])].double() * float(s["freqs"][i])
            turn = torch.polar(torch.ones_like(angle), -angle if c["backward"] else angle)
            z[:, :, i] *= turn.repeat(x.shape[0] // c["n_batch"], 1)
        out.append(torch.view_as_real(z).reshape(x.shape))
    return tuple(out)


def _sequence(s, n, pages, scales):
    """All rows that the table has for sequence n: [heads, rows, head] in 64 bits."""
    p = s["table"][n]
    p = p[p >= 0].long()
    x = pages[p].double()
    if scales is not None:
        x = x * torch.pow(2.0, scales[p].double() - 127.0)[..., None]
    return x.transpose(0, 1).reshape(pages.shape[1], -1, pages.shape[3])


def _exact_append(s):
    """What lies in the pages: for 8 bits the quotients before they are rounded."""
    c = s["case"]
    out = []
    for x, pages, scales in ((s["k"], s["k_pages"], s["k_scales"]), (s["v"], s["v_pages"], s["v_scales"])):
        now = pages.double()
        size = None if scales is None else scales.clone()
        for n in range(c["n_batch"]):
            count, length = int(s["given"][n]), int(s["lens"][n])
            position = np.arange(length - count, length)
            page = s["table"][n].long()[torch.from_numpy(position // c["page_rows"]).cuda()]
            slot = torch.from_numpy(position % c["page_rows"]).cuda()
            for hd in range(c["heads_kv"]):
                rows = x[n + c["n_batch"] * hd, :count].double()
                if scales is not None:
                    ratio = rows.abs().amax(dim=-1).cpu().numpy() / 448.0
                    k = np.array([-126 if r == 0 else max(-126, math.ceil(math.log2(r))) for r in ratio], np.int64)
                    k = torch.from_numpy(k).cuda()
                    rows = rows * torch.pow(2.0, -k.double())[:, None]
                    size[page, hd, slot] = (k + 127).to(torch.uint8)
                now[page, hd, slot] = rows
        out.append((now[:-1], None if size is None else size[:-1]))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def _exact_read(s):
    c = s["case"]
    first = c["longest"] - c["rows"]
    out = []
    for pages, scales in ((s["k_pages"], s["k_scales"]), (s["v_pages"], s["v_scales"])):
        x = torch.zeros(c["heads_kv"], c["n_batch"], c["rows"], c["head"], dtype=torch.float64, device="cuda")
        for n in range(c["n_batch"]):
            length = int(s["lens"][n])
            if length > first:
                x[:, n, :length - first] = _sequence(s, n, pages, scales)[:, first:length]
        out.append(x.reshape(-1, c["rows"], c["head"]))
    return tuple(out)


def _exact_attend(s):
    c = s["case"]
    n_batch, heads, group, rows, head = c["n_batch"], c["heads_kv"], c["kv_group"], c["rows"], c["head"]
    A = torch.zeros(heads, group, n_batch, rows, head, dtype=torch.float64, device="cuda")
    lse = torch.full((heads, group, n_batch, rows), -math.inf, dtype=torch.float64, device="cuda")
    q = s["q"].double().reshape(A.shape)
    for n in range(n_batch):
        length, count = int(s["lens"][n]), int(s["given"][n])
        k = _sequence(s, n, s["k_pages"], s["k_scales"])[:, :length].contiguous()
        v = _sequence(s, n, s["v_pages"], s["v_scales"])[:, :length].contiguous()
        for j in range(count):
            keys = length - count + j + 1
            if keys < 1:
                continue
            score = torch.matmul(q[:, :, n, j], k[:, :keys].transpose(1, 2).contiguous()) / math.sqrt(head)
            lse[:, :, n, j] = torch.logsumexp(score, dim=-1)
            A[:, :, n, j] = torch.matmul(torch.softmax(score, dim=-1), v[:, :keys].contiguous())
    return A.reshape(-1, rows, head), lse.reshape(-1, rows)
