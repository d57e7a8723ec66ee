"""Cases of a paged key/value cache for long contexts in little memory: keys and values held
in 4 bits (written, read back, attended over), the weight that each cached row has received
from attention, and the eviction of the rows that received least.

Layouts: pages [n_pages, n_head_kv, page_rows, head] (4 bits: head/2 bytes, the lower half of a
byte first); table [n_batch, max_pages] and lens [n_batch] int32 (lens counts the newest rows);
tiles [entries, rows, head] with entry = sequence + n_batch * head index; weights [n_head_kv *
n_batch, max_rows] fp32.  4-bit pages are e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), 32
neighbouring values of a row sharing a power of two that is held as its exponent + 127: the
smallest, from 2^-125 on, that leaves none of them above 7 (what rounds to the largest code is
then no further from it than half a step).  8-bit pages are e4m3 with one power of two per row.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
LARGEST = 5.4e8         # bytes of the largest listed case
CODES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _case(name, op, dtype, bits, n_batch, heads_kv, head, page_rows, longest, shortest, rows=1,
          kv_group=1, padded=False, decay=1.0, keep=0, recent=0):
    """bits: of a page's values.  longest, shortest: the lengths of the sequences run between
    the two, spread over their logarithm.  rows: new tokens a sequence.  padded: some sequences
    bring fewer tokens than that.  decay: what the weights so far are multiplied by.  keep,
    recent: rows that stay of every longer sequence, and how many of the newest are among them."""
    return {"name": name, "op": op, "dtype": dtype, "bits": bits, "n_batch": n_batch,
            "heads_kv": heads_kv, "head": head, "page_rows": page_rows, "longest": longest,
            "shortest": shortest, "rows": rows, "kv_group": kv_group, "padded": padded,
            "decay": decay, "keep": keep, "recent": recent}


def listed():
    return [
        # a generation step of eight sequences: a row a sequence and head, and what it stands for now
        _case("store_token", "store", "bf16", 4, 8, 8, 128, 64, 1001, 1001),
        # a short odd chunk of a padded batch, 12 heads of 64
        _case("store_chunk", "store", "fp16", 4, 3, 12, 64, 16, 1038, 1001, rows=77, padded=True),
        # prompts of 4096 tokens: written, and back for the products of the prompt's own attention
        _case("store_prompt", "store", "bf16", 4, 4, 8, 128, 64, 4096, 4096, rows=4096),
        # one user's generation step at a short context: latency
        _case("attend_one_user", "attend", "bf16", 4, 1, 8, 128, 64, 1001, 1001, kv_group=4),
        # four drafted tokens to check, fewer in some of the sequences, 8 query heads on one
        _case("attend_drafts", "attend", "fp16", 4, 16, 8, 64, 64, 4096, 300, rows=4, kv_group=8,
              padded=True),
        # serving: 64 sequences of 17 to 16384 tokens in pages of 16 rows
        _case("attend_ragged", "attend", "bf16", 4, 64, 8, 128, 16, 16384, 17, kv_group=4),
        # the decode workload: 16 new tokens over 8192, 32 query heads on 8
        _case("attend_decode", "attend", "bf16", 4, 8, 8, 128, 128, 8192, 8192, rows=16, kv_group=4),
        # a generation step's weights, eight sequences of 500 to 8192 rows, older steps fading
        _case("weights_token", "weights", "bf16", 16, 8, 8, 128, 64, 8192, 500, kv_group=4, decay=0.95),
        # the last 32 queries of four prompts say which of their rows matter; 4-bit rows
        _case("weights_window", "weights", "fp16", 4, 4, 8, 128, 64, 4096, 4096, rows=32, kv_group=4,
              decay=0.0),
        # a small fp32 model, one sequence of 1024 rows: half of them go
        _case("evict_small_fp32", "evict", "fp32", 32, 1, 12, 64, 32, 1024, 1024, keep=512, recent=64),
        # eight prompts in 4 bits of 700 to 8192 rows, 1024 stay, and what they stand for
        _case("evict_prompt", "evict", "bf16", 4, 8, 8, 128, 64, 8192, 700, keep=1024, recent=128),
        # a full cache makes room for the next page of every sequence: nearly all rows stay
        _case("evict_page", "evict", "bf16", 16, 8, 8, 128, 64, 8192, 8192, keep=8128, recent=512),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["store", "attend", "attend", "weights", "evict"])
        bits = 4 if op in ("store", "attend") else rng.choice([4, 8, 16, 16, 32])
        dtype = "fp32" if bits == 32 else rng.choice(["bf16", "fp16"])
        head = rng.choice([64, 128])
        n_batch = _log(rng, 1, 64)
        longest = _log(rng, 1, 16384)
        shortest = longest if rng.random() < 0.4 else _log(rng, 1, longest)
        most = {"store": shortest, "attend": min(16, shortest), "weights": min(64, shortest), "evict": 1}[op]
        rows = 1 if rng.random() < 0.3 else _log(rng, 1, most)
        keep = _log(rng, 1, longest) if op == "evict" else 0
        c = _case("", op, dtype, bits, n_batch, rng.choice([1, 2, 4, 8, 12, 16]), head,
                  rng.choice([16, 32, 64, 128, 256]), longest, shortest, rows=rows,
                  kv_group=rng.choice([1, 1, 2, 4, 8]) if op in ("attend", "weights") else 1,
                  padded=op != "evict" and rng.random() < 0.3,
                  decay=rng.choice([0.0, 0.9, 1.0]) if op == "weights" else 1.0,
                  keep=keep, recent=rng.randrange(0, keep + 1) if keep else 0)
        if work(c)["bytes"] <= LARGEST and _plain_bytes(c) <= 1.2e10 and _pool_bytes(c) <= 1.2e9:
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


def _stored(case):
    """Bytes of a row of keys, or of values, in its page."""
    head = case["head"]
    return {4: head // 2 + head // 32, 8: head + 1}.get(case["bits"], head * BYTES[case["dtype"]])


def _span(case):
    """The rows that are read back: (first, number)."""
    if case["op"] == "evict":
        return 0, min(case["keep"], case["longest"])
    first = case["shortest"] - case["rows"]
    return first, case["longest"] - first


def _pool_bytes(case):
    pages = sum(-(-l // case["page_rows"]) for l in _lens(case))
    return 2.0 * pages * case["page_rows"] * case["heads_kv"] * case["head"] * 4


def _plain_bytes(case):
    """What the plain form holds at most: padded fp32 copies of keys and values."""
    rows = case["rows"] * case["kv_group"] if case["op"] in ("attend", "weights") else 0
    return 8.0 * case["n_batch"] * case["heads_kv"] * case["longest"] * (case["head"] + rows)


def _read_bytes(case):
    first, rows = _span(case)
    there = sum(min(max(0, l - first), rows) for l in _lens(case)) * case["heads_kv"]
    out = case["n_batch"] * case["heads_kv"] * rows * case["head"] * BYTES[case["dtype"]]
    return 2 * (there * _stored(case) + out)


def work(case):
    e, head, heads = BYTES[case["dtype"]], case["head"], case["heads_kv"]
    lens, stored = _lens(case), _stored(case)
    if case["op"] in ("attend", "weights"):
        rows, group = case["rows"], case["kv_group"]
        queries = case["n_batch"] * heads * group * rows
        pairs = sum(new * l - new * (new - 1) // 2 for l, new in zip(lens, _new_rows(case))) * heads * group
        if case["op"] == "attend":
            return {"bytes": 2 * sum(lens) * heads * stored + queries * (2 * head * e + 4), "flops": 4 * pairs * head}
        old = 4 if case["decay"] else 0
        return {"bytes": sum(lens) * heads * (stored + 4 + old) + queries * (head * e + 4), "flops": 2 * pairs * head}
    if case["op"] == "store":
        moved = sum(_new_rows(case)) * heads
        return {"bytes": 2 * moved * (head * e + stored) + _read_bytes(case), "flops": 4 * moved * head}
    keep, recent = case["keep"], case["recent"]
    bytes_, kept = 0, 0
    for l in lens:
        stay = min(l, keep)
        kept += stay
        # a row read and written again for every one behind the first that goes
        moved = keep - (l - recent + 1) // (l - keep + 1) if l > keep else 0
        bytes_ += 8 * l + 4 * stay + 4 * stored * max(0, moved)
    return {"bytes": heads * bytes_ + (_read_bytes(case) if case["bits"] == 4 else 0), "flops": heads * (sum(lens) + kept)}


def _codes4(x):
    """Blocks of 32 values of the last axis as codes (two a byte) and scale bytes."""
    b = x.float().reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    mantissa, exponent = torch.frexp(b.abs().amax(dim=-1))
    # 7 = 0.875 * 2^3
    k = torch.where(mantissa > 0.875, exponent - 2, exponent - 3).clamp(min=-125)
    k = torch.where(mantissa == 0, -125, k)
    y = torch.ldexp(b, -k[..., None])
    size = y.abs()
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    size = (torch.round(size / step) * step).clamp(max=6.0)
    code = torch.where(size <= 2, 2 * size, torch.where(size <= 4, size + 2, size / 2 + 4)).to(torch.uint8)
    code = (code + 8 * torch.signbit(y).to(torch.uint8)).reshape(*x.shape[:-1], x.shape[-1] // 2, 2)
    return code[..., 0] + 16 * code[..., 1], (k + 127).to(torch.uint8)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = TYPES[case["dtype"]]
    head, n_batch, heads, page_rows = case["head"], case["n_batch"], case["heads_kv"], case["page_rows"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).to(dt)

    def whole(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=gen, device="cuda")

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
    k_scales = v_scales = None
    if case["bits"] == 4:
        # codes of all kinds, values of about the size of normal ones
        k_pages, v_pages = (whole(0, 256, *shape[:3], head // 2).to(torch.uint8) for _ in range(2))
        k_scales, v_scales = (whole(125, 127, *shape[:3], head // 32).to(torch.uint8) for _ in range(2))
    elif case["bits"] == 8:
        k_pages, v_pages = ((3e2 * torch.rand(shape, generator=gen, device="cuda") - 150.0).to(torch.float8_e4m3fn)
                            for _ in range(2))
        k_scales, v_scales = (whole(119, 122, *shape[:3]).to(torch.uint8) for _ in range(2))
    else:
        k_pages, v_pages = normal(*shape), normal(*shape)
    s = {"case": case, "k_pages": k_pages, "v_pages": v_pages, "k_scales": k_scales, "v_scales": v_scales,
         "table": table, "lens": lens, "new_rows": new_rows if case["padded"] else None, "given": new_rows}
    entries, rows = n_batch * heads, case["rows"]
    max_rows = max_pages * page_rows
    if case["op"] == "store":
        s["k"], s["v"] = normal(entries, rows, head), normal(entries, rows, head)
    if case["op"] == "store" or (case["op"] == "evict" and case["bits"] == 4):
        s["k_out"] = torch.empty(entries, _span(case)[1], head, dtype=dt, device="cuda")
        s["v_out"] = torch.empty_like(s["k_out"])
    if case["op"] in ("attend", "weights"):
        s["q"] = normal(entries * case["kv_group"], rows, head)
        s["A"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(entries * case["kv_group"], rows, dtype=torch.float32, device="cuda")
        # memory for what the shares of a long cache leave for each other, kept between steps
        s["workspace"] = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    if case["op"] == "weights":
        s["lse"] = _plain_attend(s, only_lse=True)
    if case["op"] in ("weights", "evict"):
        # a few rows have most of the weight, some have none yet
        w = torch.exp(2.0 * torch.randn(entries, max_rows, generator=gen, device="cuda") - 4.0)
        w *= torch.rand(entries, max_rows, generator=gen, device="cuda") > 0.1
        s["weights"] = torch.where(torch.arange(max_rows, device="cuda") < lens.repeat(heads)[:, None], w, 0.0)
    if case["op"] == "evict":
        s["weights_out"] = torch.zeros_like(s["weights"])
        s["kept"] = torch.full((entries, case["keep"]), -1, dtype=torch.int32, device="cuda")
        s["lens_after"] = lens.clamp(max=case["keep"])
    return s


def run(s):
    if own:
        return _run_own(s)
    return {"store": _plain_store, "attend": _plain_attend, "weights": _plain_weights, "evict": _plain_evict}[s["case"]["op"]](s)


def _run_own(s):
    from nntile_amd import hip_sdpa as h
    c = s["case"]
    k_pages, v_pages, k_scales, v_scales = s["k_pages"][:-1], s["v_pages"][:-1], None, None
    if c["bits"] <= 8:
        k_scales, v_scales = s["k_scales"][:-1], s["v_scales"][:-1]
    if c["bits"] == 4:
        k_pages, v_pages = k_pages.view(torch.float4_e2m1fn_x2), v_pages.view(torch.float4_e2m1fn_x2)
    if c["op"] == "store":
        h.paged_kv_append(s["k"], s["v"], k_pages, v_pages, s["table"], s["lens"], k_scales, v_scales,
                          new_rows=s["new_rows"])
        h.paged_kv_read(k_pages, v_pages, s["table"], s["lens"], s["k_out"], s["v_out"], first=_span(c)[0],
                        k_scales=k_scales, v_scales=v_scales)
        return s["k_out"], s["v_out"]
    if c["op"] == "attend":
        h.sdpa_fwd_paged(k_pages, v_pages, s["table"], s["lens"], s["q"], s["lse"], s["A"], h.MASK_CAUSAL,
                         c["kv_group"], s["workspace"], k_scales=k_scales, v_scales=v_scales,
                         new_rows=s["new_rows"], flags=h.OVERWRITE)
        return s["A"], s["lse"]
    if c["op"] == "weights":
        h.paged_attn_weights(k_pages, s["table"], s["lens"], s["q"], s["lse"], s["weights"], h.MASK_CAUSAL,
                             c["kv_group"], k_scales=k_scales, new_rows=s["new_rows"], decay=c["decay"])
        return s["weights"]
    h.paged_kv_evict(k_pages, v_pages, s["table"], s["lens"], s["weights"], s["weights_out"], s["kept"],
                     c["recent"], k_scales=k_scales, v_scales=v_scales)
    if c["bits"] == 4:
        h.paged_kv_read(k_pages, v_pages, s["table"], s["lens_after"], s["k_out"], s["v_out"],
                        k_scales=k_scales, v_scales=v_scales)
        return s["kept"], s["weights_out"], s["k_out"], s["v_out"]
    return s["kept"], s["weights_out"], k_pages, v_pages, k_scales, v_scales


# ---- plain forms: elementary torch operations in 32 bits -------------------------

def _rows_of(s, position, wanted):
    """The flat page rows of every head's row at `position`, [n_batch, positions] or [n_batch,
    heads, positions]; the spare page's where `wanted` is false."""
    c = s["case"]
    page_rows, heads = c["page_rows"], c["heads_kv"]
    if position.dim() == 2:
        position, wanted = (x[:, None, :].expand(-1, heads, -1) for x in (position, wanted))
    slot = (position // page_rows).clamp(0, s["table"].shape[1] - 1)
    page = torch.gather(s["table"].long()[:, None, :].expand(-1, heads, -1), 2, slot)
    page = torch.where(wanted, page, s["k_pages"].shape[0] - 1)
    head = torch.arange(heads, device="cuda")[None, :, None]
    return (page * heads + head) * page_rows + position % page_rows


def _plain_rows(s, pages, scales, at):
    """The page rows `at`, as fp32 values."""
    c = s["case"]
    x = pages.view(-1, pages.shape[-1])
    if c["bits"] == 4:
        code = torch.stack((x[at] & 15, x[at] >> 4), dim=-1).long()
        sign = 1 - 2 * (code >> 3)
        code = torch.tensor(CODES, device="cuda")[code & 7] * sign
        code = code.reshape(*at.shape, c["head"] // 32, 32)
        size = scales.view(-1, c["head"] // 32)[at].int() - 127
        return torch.ldexp(code, size[..., None]).reshape(*at.shape, c["head"])
    if c["bits"] == 8:
        code = x.view(torch.uint8)[at].view(torch.float8_e4m3fn).float()
        return torch.ldexp(code, scales.view(-1)[at].int()[..., None] - 127)
    return x[at].float()


def _plain_read(s, lens):
    c = s["case"]
    first, rows = _span(c)
    position = torch.arange(first, first + rows, device="cuda")[None, :].expand(c["n_batch"], rows)
    there = position < lens[:, None]
    at = _rows_of(s, position, there)
    out = []
    for pages, scales in ((s["k_pages"], s["k_scales"]), (s["v_pages"], s["v_scales"])):
        x = torch.where(there[:, None, :, None], _plain_rows(s, pages, scales, at), 0.0)
        out.append(x.transpose(0, 1).reshape(-1, rows, c["head"]).to(TYPES[c["dtype"]]))
    return tuple(out)


def _plain_store(s):
    c = s["case"]
    n_batch, heads, head, rows = c["n_batch"], c["heads_kv"], c["head"], c["rows"]
    r = torch.arange(rows, device="cuda")[None, :]
    new = s["given"][:, None]
    at = _rows_of(s, (s["lens"][:, None] - new + r).clamp(min=0), r < new).reshape(-1)
    for x, pages, scales in ((s["k"], s["k_pages"], s["k_scales"]), (s["v"], s["v_pages"], s["v_scales"])):
        codes, size = _codes4(x.reshape(heads, n_batch, rows, head).transpose(0, 1).reshape(-1, head))
        pages.view(-1, head // 2)[at] = codes
        scales.view(-1, head // 32)[at] = size
    return _plain_read(s, s["lens"])


def _scores(s):
    """Scores [n_batch, heads, group * rows, longest], -inf where a query does not see the row."""
    c = s["case"]
    n_batch, heads, head, rows, group = c["n_batch"], c["heads_kv"], c["head"], c["rows"], c["kv_group"]
    position = torch.arange(c["longest"], device="cuda")[None, :].expand(n_batch, c["longest"])
    there = position < s["lens"][:, None]
    at = _rows_of(s, position, there)
    k = _plain_rows(s, s["k_pages"], s["k_scales"], at)                # [n_batch, heads, longest, head]
    q = s["q"].float().reshape(heads, group, n_batch, rows, head).permute(2, 0, 1, 3, 4)
    q = q.reshape(n_batch, heads, group * rows, head)
    score = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(head))
    j = torch.arange(rows, device="cuda")
    last = s["lens"][:, None] - s["given"][:, None] + j                # the last row a query sees
    seen = (position[:, None, :] <= last[:, :, None]) & (j < s["given"][:, None])[:, :, None] & there[:, None, :]
    seen = seen[:, None, None].expand(n_batch, heads, group, rows, c["longest"]).reshape(score.shape)
    return torch.where(seen, score, -math.inf), there, at


def _plain_attend(s, only_lse=False):
    c = s["case"]
    n_batch, heads, rows, group = c["n_batch"], c["heads_kv"], c["rows"], c["kv_group"]
    score, there, at = _scores(s)
    top = score.amax(dim=-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    weight = torch.exp(score - top)
    total = weight.sum(dim=-1, keepdim=True)
    lse = torch.log(total) + top

    def back(x):
        x = x.reshape(n_batch, heads, group, rows, x.shape[-1]).permute(1, 2, 0, 3, 4)
        return x.reshape(heads * group * n_batch, rows, x.shape[-1])

    if only_lse:
        return back(lse).squeeze(-1).contiguous()
    v = torch.where(there[:, None, :, None], _plain_rows(s, s["v_pages"], s["v_scales"], at), 0.0)
    A = torch.matmul(weight, v) / torch.where(total == 0, 1.0, total)
    return back(A).to(TYPES[c["dtype"]]), back(lse).squeeze(-1)


def _plain_weights(s):
    c = s["case"]
    n_batch, heads, rows, group = c["n_batch"], c["heads_kv"], c["rows"], c["kv_group"]
    score, there, _ = _scores(s)
    lse = s["lse"].reshape(heads, group, n_batch, rows).permute(2, 0, 1, 3).reshape(n_batch, heads, group * rows, 1)
    weight = torch.where(score == -math.inf, 0.0, torch.exp(score - lse)).sum(dim=2)       # [n_batch, heads, longest]
    weight = weight.transpose(0, 1).reshape(heads * n_batch, -1)
    there = there[None].expand(heads, -1, -1).reshape(heads * n_batch, -1)
    so_far = s["weights"][:, :c["longest"]]
    so_far.copy_(torch.where(there, weight + (so_far * c["decay"] if c["decay"] else 0.0), so_far))
    return s["weights"]


def _plain_evict(s):
    c = s["case"]
    n_batch, heads, keep, longest = c["n_batch"], c["heads_kv"], c["keep"], c["longest"]
    keep_here = min(keep, longest)
    lens = s["lens"].long()[:, None, None]
    position = torch.arange(longest, device="cuda")[None, None, :].expand(n_batch, heads, longest)
    w = s["weights"][:, :longest].reshape(heads, n_batch, longest).transpose(0, 1)
    rank = torch.where(position >= lens, -math.inf, torch.where(position >= lens - c["recent"], math.inf, w))
    # the heaviest first, of equal ones the lower row
    best = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep_here]
    best = torch.sort(torch.where(best < lens, best, longest), dim=-1).values
    there = best < lens
    src = _rows_of(s, torch.where(there, best, 0), there).reshape(-1)
    dst = _rows_of(s, position[..., :keep_here], there).reshape(-1)
    for pages, scales in ((s["k_pages"], s["k_scales"]), (s["v_pages"], s["v_scales"])):
        for x in (pages, scales):
            if x is not None:
                x = x.view(torch.uint8) if x.element_size() == 1 else x
                x = x.view(-1, 1) if c["bits"] == 8 and x.dim() == 3 else x.view(-1, x.shape[-1])
                x[dst] = x[src]

    def entries(x):
        return x.transpose(0, 1).reshape(heads * n_batch, -1)

    s["kept"][:, :keep_here] = entries(torch.where(there, best, -1)).to(torch.int32)
    s["kept"][:, keep_here:] = -1
    moved = torch.zeros_like(w)
    moved[..., :keep_here] = torch.where(there, torch.gather(w, 2, torch.where(there, best, 0)), 0.0)
    out = s["weights_out"][:, :longest]
    out.copy_(torch.where(entries(position < lens), entries(moved), out))
    if c["bits"] == 4:
        return (s["kept"], s["weights_out"]) + _plain_read(s, s["lens_after"])
    scales = (None, None) if c["bits"] > 8 else (s["k_scales"][:-1], s["v_scales"][:-1])
    return (s["kept"], s["weights_out"], s["k_pages"][:-1], s["v_pages"][:-1]) + scales


# ---- the operators' definitions in 64 bits ----------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"store": _exact_store, "attend": _exact_attend, "weights": _exact_weights, "evict": _exact_evict}[case["op"]](s)


def _values(s, pages, scales):
    """All values of the pool in 64 bits."""
    if s["case"]["bits"] == 4:
        value = torch.tensor(CODES + tuple(-x for x in CODES), dtype=torch.float64, device="cuda")
        x = torch.empty(pages.shape[:-1] + (s["case"]["head"],), dtype=torch.float64, device="cuda")
        x[..., 0::2] = value[pages.long() % 16]
        x[..., 1::2] = value[pages.long() // 16]
        return x * torch.pow(2.0, scales.double() - 127.0).repeat_interleave(32, dim=-1)
    x = pages.double()
    return x if scales is None else x * torch.pow(2.0, scales.double() - 127.0)[..., None]


def _sequence(s, n, pool):
    """All rows that the table has for sequence n: [heads, rows, head] in 64 bits."""
    p = s["table"][n]
    x = pool[p[p >= 0].long()]
    return x.transpose(0, 1).reshape(pool.shape[1], -1, pool.shape[3])


def _rounded4(x):
    """Values [.., 32], in numpy, as the nearest of the codes times the block's power of two."""
    out = np.zeros_like(x)
    top = np.abs(x).max(axis=-1)
    k = np.where(top == 0, -125, np.maximum(-125, np.ceil(np.log2(np.where(top == 0, 1.0, top) / 7.0))))
    y = np.abs(x) * np.exp2(-k)[..., None]
    grid = np.array(CODES)
    middle = (grid[1:] + grid[:-1]) / 2
    at = np.searchsorted(middle, y, side="left")        # of two equally near ones the lower ...
    tie = (at < 7) & (middle[np.minimum(at, 6)] == y)
    at = np.where(tie & (at % 2 == 1), at + 1, at)      # ... unless its last bit is set
    out = np.copysign(grid[at], x) * np.exp2(k)[..., None]
    return out


def _exact_store(s):
    c = s["case"]
    first, rows = _span(c)
    out = []
    for x, pages, scales in ((s["k"], s["k_pages"], s["k_scales"]), (s["v"], s["v_pages"], s["v_scales"])):
        pool = _values(s, pages, scales)
        new = x.double().cpu().numpy()
        new = torch.from_numpy(_rounded4(new.reshape(-1, c["head"] // 32, 32)).reshape(new.shape)).cuda()
        new = new.reshape(c["heads_kv"], c["n_batch"], c["rows"], c["head"])
        got = torch.zeros(c["heads_kv"], c["n_batch"], rows, c["head"], dtype=torch.float64, device="cuda")
        for n in range(c["n_batch"]):
            count, length = int(s["given"][n]), int(s["lens"][n])
            now = _sequence(s, n, pool)
            now[:, length - count:length] = new[:, n, :count]
            got[:, n, :length - first] = now[:, first:length]
        out.append(got.reshape(-1, rows, c["head"]))
    return tuple(out)


def _exact_attend(s):
    c = s["case"]
    n_batch, heads, group, rows, head = c["n_batch"], c["heads_kv"], c["kv_group"], c["rows"], c["head"]
    A = torch.zeros(heads, group, n_batch, rows, head, dtype=torch.float64, device="cuda")
    lse = torch.full((heads, group, n_batch, rows), -math.inf, dtype=torch.float64, device="cuda")
    q = s["q"].double().reshape(A.shape)
    keys, values = _values(s, s["k_pages"], s["k_scales"]), _values(s, s["v_pages"], s["v_scales"])
    for n in range(n_batch):
        length, count = int(s["lens"][n]), int(s["given"][n])
        k = _sequence(s, n, keys)[:, :length].contiguous()
        v = _sequence(s, n, values)[:, :length].contiguous()
        for j in range(count):
            seen = length - count + j + 1
            if seen < 1:
                continue
            score = torch.matmul(q[:, :, n, j], k[:, :seen].transpose(1, 2).contiguous()) / math.sqrt(head)
            lse[:, :, n, j] = torch.logsumexp(score, dim=-1)
            A[:, :, n, j] = torch.matmul(torch.softmax(score, dim=-1), v[:, :seen].contiguous())
    return A.reshape(-1, rows, head), lse.reshape(-1, rows)


def _exact_weights(s):
    c = s["case"]
    n_batch, heads, group, rows, head = c["n_batch"], c["heads_kv"], c["kv_group"], c["rows"], c["head"]
    out = s["weights"].double().reshape(heads, n_batch, -1)
    q = s["q"].double().reshape(heads, group, n_batch, rows, head)
    lse = s["lse"].double().reshape(heads, group, n_batch, rows)
    keys = _values(s, s["k_pages"], s["k_scales"])
    for n in range(n_batch):
        length, count = int(s["lens"][n]), int(s["given"][n])
        k = _sequence(s, n, keys)[:, :length].transpose(1, 2).contiguous()
        out[:, n, :length] *= c["decay"]
        for j in range(count):
            seen = length - count + j + 1
            score = torch.matmul(q[:, :, n, j], k[:, :, :seen].contiguous()) / math.sqrt(head)
            out[:, n, :seen] += torch.exp(score - lse[:, :, n, j, None]).sum(dim=1)
    return out.reshape(heads * n_batch, -1)


def _exact_evict(s):
    c = s["case"]
    n_batch, heads, keep, recent, page_rows = c["n_batch"], c["heads_kv"], c["keep"], c["recent"], c["page_rows"]
    weights, out = s["weights"].double().cpu().numpy(), s["weights_out"].double().cpu().numpy()
    kept = np.full((heads * n_batch, keep), -1, np.int32)
    pools = [x[:-1].double() if c["bits"] != 4 else _values(s, x, y)[:-1]
             for x, y in ((s["k_pages"], s["k_scales"]), (s["v_pages"], s["v_scales"]))]
    sizes = [x[:-1].clone() if c["bits"] == 8 else None for x in (s["k_scales"], s["v_scales"])]
    for n in range(n_batch):
        length = int(s["lens"][n])
        pages = s["table"][n].long()
        for hd in range(heads):
            e = n + n_batch * hd
            w = weights[e, :length]
            old = max(0, length - recent)
            stay = np.arange(length)
            if length > keep:
                by_weight = np.lexsort((np.arange(old), -w[:old]))
                stay = np.sort(np.concatenate((by_weight[:keep - (length - old)], np.arange(old, length))))
            kept[e, :len(stay)] = stay
            out[e, :length] = 0.0
            out[e, :len(stay)] = w[stay]
            src = torch.from_numpy(stay).cuda()
            dst = torch.arange(len(stay), device="cuda")
            for pool in pools + [x for x in sizes if x is not None]:
                pool[pages[dst // page_rows], hd, dst % page_rows] = pool[pages[src // page_rows], hd, src % page_rows]
    kept, out = torch.from_numpy(kept).cuda(), torch.from_numpy(out).cuda()
    if c["bits"] != 4:
        return (kept, out) + tuple(pools) + tuple(sizes)
    rows = _span(c)[1]
    tiles = []
    for pool in pools:
        x = torch.zeros(heads, n_batch, rows, c["head"], dtype=torch.float64, device="cuda")
        for n in range(n_batch):
            there = min(int(s["lens"][n]), rows)
            x[:, n, :there] = _sequence(s, n, pool)[:, :there]
        tiles.append(x.reshape(-1, rows, c["head"]))
    return (kept, out) + tuple(tiles)
