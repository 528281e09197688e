"""Operators of a serving step with several continuations of a prompt, over a paged cache held in 4 bits, as cases that can be timed.

  write    `tpa_cache_write_fp4` and `tpa_cache_read_fp4`: the K and V factors of new tokens into their slots of a paged cache of 4-bit codes with
           a scale for each 32 of them, and the values that the slots then hold
  decode   `tpa_decode_fp4`: a few query tokens of every sequence over such a cache
  select   `tpa_beam_select`: the best continuations over the beams and the vocabulary
  fork     `tpa_pages_fork`: sequences that go on from chosen ones: pages shared, the last one copied, those of dropped sequences released
  compact  `tpa_pages_compact`: pages moved to the front of their pools

With `own` false the same is computed in its plain form by elementary torch operations.
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
PAGE = 64
EOS = 2
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # what the codes 0 .. 7 stand for; 8 .. 15 are their negatives


def listed():
    return [
        # the new tokens of a decode step of 48 conversations
        dict(name="write_step", kind="write", T=48, H=32, D=128, rk=2, dtype="bf16"),
        # a step's packed chunk of prompts, a number of tokens that is no round one
        dict(name="write_chunk", kind="write", T=8195, H=32, D=128, rk=2, dtype="bf16"),
        # four continuations of a user's prompt, a small model
        dict(name="decode_few", kind="decode", B=4, lq=1, keys=1500, H=16, D=128, rq=6, rk=2, dtype="bf16"),
        # a full server with caches of up to 12 000 tokens
        dict(name="decode_batch", kind="decode", B=128, lq=1, keys=12000, H=32, D=128, rq=6, rk=2, dtype="bf16"),
        # speculated tokens, verified in one step, narrow heads and a higher rank
        dict(name="decode_speculative", kind="decode", B=12, lq=4, keys=4500, H=64, D=64, rq=6, rk=4, dtype="bf16"),
        # queries in the reference's default type
        dict(name="decode_f32", kind="decode", B=8, lq=1, keys=2200, H=8, D=64, rq=6, rk=2, dtype="f32"),
        # one user's beams, logits in 32 bits, a vocabulary of an odd size
        dict(name="select_few", kind="select", B=1, beams=4, vocab=50021, dtype="f32"),
        # a server's requests with four beams each, a large vocabulary, logits as a 16-bit model gives them
        dict(name="select_batch", kind="select", B=64, beams=4, vocab=131072, dtype="bf16"),
        # the step after select_few: one user's beams over the caches of four layers
        dict(name="fork_few", kind="fork", B=1, beams=4, cache=1500, layers=4, H=16, D=128, rk=2),
        # that of a server: requests that end beside others that go on
        dict(name="fork_batch", kind="fork", B=64, beams=4, cache=4096, layers=8, H=32, D=128, rk=2),
        # a small server's pools after its last requests ended, few pages free
        dict(name="compact_few", kind="compact", B=6, cache=2000, holes=0.1, layers=2, H=16, D=64, rk=2),
        # pools with holes all over them are made dense before a part of them is given away
        dict(name="compact_batch", kind="compact", B=96, cache=4096, holes=0.3, layers=8, H=32, D=128, rk=2),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _cost(case):
    w = work(case)
    return w["flops"] / (2e14 if case.get("dtype", "bf16") == "bf16" else 4e13) + w["bytes"] / 4e12


def draw(rng):
    limit = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(["write", "decode", "decode", "select", "fork", "compact"])
        h, d = rng.choice([(8, 64), (16, 64), (64, 64), (16, 128), (32, 128), (24, 128)])
        rk = rng.choice([1, 2, 2, 4, 8])
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        if kind == "write":
            case = dict(kind=kind, T=_log_int(rng, 1, 16384), H=h, D=d, rk=rk, dtype=dtype)
        elif kind == "decode":
            case = dict(kind=kind, B=_log_int(rng, 1, 160), lq=rng.choice([1, 1, 1, 2, 5]), keys=_log_int(rng, 16, 40000), H=h, D=d, rq=rng.choice([1, 3, 6, 16]), rk=rk, dtype=dtype)
        elif kind == "select":
            case = dict(kind=kind, B=_log_int(rng, 1, 96), beams=rng.choice([1, 2, 3, 4, 5, 8, 16]), vocab=_log_int(rng, 500, 160000), dtype=dtype)
            if case["B"] * case["beams"] * case["vocab"] > 3.5e7:
                continue
        elif kind == "fork":
            case = dict(kind=kind, B=_log_int(rng, 1, 96), beams=rng.choice([2, 3, 4, 5, 8]), cache=_log_int(rng, 100, 8192), layers=rng.randint(1, 8), H=h, D=d, rk=rk)
        else:
            case = dict(kind=kind, B=_log_int(rng, 1, 96), cache=_log_int(rng, 200, 8192), holes=round(rng.uniform(0.02, 0.6), 2), layers=rng.randint(1, 8), H=h, D=d, rk=rk)
        if _cost(case) <= limit and _pool_bytes(case) < 4e9:
            return case


# ---------------------------------------------------------------------------------------------- sizes
def _row(h, d):
    """Bytes of a rank's row: codes of d and of h values, a scale for each 32 of either, up to a multiple of four."""
    return -(-((d + 1) // 2 + (h + 1) // 2 + -(-d // 32) + -(-h // 32)) // 4) * 4


def _own_keys(case):
    """Keys of each sequence, the new tokens among them: from a half to all of `keys`; the same for all seeds but in order."""
    keys = case["keys"]
    return [max(case["lq"], keys - (i * 7919) % (keys // 2 + 1)) for i in range(case["B"])]


def _group(case, i):
    """Length of request i's beams and the tokens that they share."""
    length = max(2, case["cache"] - (i * 7919) % (case["cache"] // 2 + 1))
    return length, length - min(length - 1, 17 + (i * 31) % 150)


def _parents(case, i):
    """Beam that each of request i's next beams goes on from: beams that are picked twice and more, beams that nobody picks; None: the request ends."""
    if i % 8 == 5:
        return None
    return [(j * (j + 2 + i) // 2) % case["beams"] for j in range(case["beams"])]


def _fork_sizes(case):
    """(tokens copied, pages of all beams together, pages in a row of the table, table entries in use)"""
    copied = pages = most = entries = 0
    for i in range(case["B"]):
        length, shared = _group(case, i)
        each, in_common = -(-length // PAGE), shared // PAGE
        pages += in_common + case["beams"] * (each - in_common)
        most = max(most, each)
        entries += each * case["beams"]
        found = _parents(case, i)
        if found is not None:
            copied += (length % PAGE) * (len(found) - len(set(found)))
    return copied, pages, most + 1, entries


def _compact_sizes(case):
    """(pages in use, of all pages)"""
    used = sum(-(-_group(case, i)[0] // PAGE) for i in range(case["B"]))
    return used, used + max(1, round(used * case["holes"] / (1 - case["holes"])))


def _pool_bytes(case):
    if case["kind"] not in ("fork", "compact"):
        return 0
    pages = _fork_sizes(case)[1] + 2 * case["B"] * case["beams"] + 8 if case["kind"] == "fork" else _compact_sizes(case)[1]
    return pages * PAGE * case["rk"] * _row(case["H"], case["D"]) * 2 * case["layers"]


def work(case):
    if case["kind"] == "select":
        n = case["B"] * case["beams"]
        return {"bytes": n * case["vocab"] * (2 if case["dtype"] == "bf16" else 4) + n * (4 + 1 + 4 + 4 + 4 + 1), "flops": 6 * n * case["vocab"]}
    h, d, rk = case["H"], case["D"], case["rk"]
    token = 2 * rk * _row(h, d)  # of a cached token, K and V
    if case["kind"] == "write":
        e = 2 if case["dtype"] == "bf16" else 4
        # factors read, rows written; rows read, values written
        return {"bytes": case["T"] * (2 * e * 2 * rk * (h + d) + 2 * token + 8), "flops": case["T"] * 2 * rk * (h + d) * 4}
    if case["kind"] == "decode":
        e = 2 if case["dtype"] == "bf16" else 4
        tokens, rows = sum(_own_keys(case)), case["B"] * case["lq"] * h
        return {"bytes": tokens * token + 4 * tokens // PAGE + rows // h * case["rq"] * (h + d) * e + rows * (d * e + 4), "flops": 4 * d * rk * case["lq"] * h * tokens}
    if case["kind"] == "fork":
        copied, pages, _, entries = _fork_sizes(case)
        rows = case["B"] * case["beams"]
        pages += 2 * rows + 8
        # contents copied; tables, lengths, parents, shares and free pages read and written
        return {"bytes": 2 * copied * token * case["layers"] + 8 * entries + 12 * rows + 16 * pages, "flops": pages + entries}
    used, pages = _compact_sizes(case)
    moved = used * (pages - used) // pages  # on average
    return {"bytes": 2 * moved * PAGE * token * case["layers"] + 8 * used + 16 * pages, "flops": pages + used}


# ---------------------------------------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _bytes(g, *shape):
    return torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.uint8)


def prepare(case, seed):
    g = _generator(seed)
    s = dict(case)
    order = torch.Generator().manual_seed(seed)
    if case["kind"] == "select":
        b, n, vocab = case["B"], case["beams"], case["vocab"]
        s["logits"] = _normal(g, b, n, vocab, dtype=DTYPES[case["dtype"]], scale=2.5)
        s["scores"] = -10 * torch.rand(b, n, generator=g, device="cuda")
        s["finished"] = torch.rand(b, n, generator=g, device="cuda") < 0.1
        return s
    h, d, rk = (case[k] for k in ("H", "D", "rk"))
    row = _row(h, d)
    if case["kind"] == "write":
        tokens, dtype = case["T"], DTYPES[case["dtype"]]
        rows = -(-tokens // 16) * 16  # a step's rows are padded
        n_pages = rows // PAGE + 9
        s["k"], s["v"] = (_normal(g, 1, rows, rk, h + d, dtype=dtype) for _ in range(2))
        s["slots"] = torch.randperm(n_pages * PAGE, generator=g, device="cuda")[:rows].to(torch.int32).view(1, rows).contiguous()
        s["slots"][:, tokens:] = -1
        s["pools"] = [torch.zeros((n_pages, PAGE, rk, row), dtype=torch.uint8, device="cuda") for _ in range(2)]
        return s
    if case["kind"] == "decode":
        # factors whose queries and keys have a root mean square of one, as norms leave them
        b, lq = case["B"], case["lq"]
        lengths = torch.tensor(_own_keys(case), dtype=torch.int32)[torch.randperm(b, generator=order)]
        pages = -(-case["keys"] // PAGE)
        s["q"] = _normal(g, b, lq, case["rq"], h + d, dtype=DTYPES[case["dtype"]])
        s["q"][..., :h] *= case["rq"] ** 0.5
        s["table"] = torch.randperm(b * pages, generator=g, device="cuda").to(torch.int32).view(b, pages)
        s["pools"] = [torch.empty((b * pages, PAGE, rk, row), dtype=torch.uint8, device="cuda") for _ in range(2)]
        for pool, scale in zip(s["pools"], (rk**0.5, 1.0)):
            for part in pool.split(2048):
                x = _normal(g, *part.shape[:3], h + d)
                x[..., :h] *= scale
                part.copy_(_plain_rows(x, h))
        s["lengths"] = lengths.cuda()
        return s
    page_bytes = (PAGE, rk, row)
    if case["kind"] == "fork":
        b, n = case["B"], case["beams"]
        _, in_use, per_row, _ = _fork_sizes(case)
        total = in_use + 2 * b * n + 8
        ids = torch.randperm(total, generator=order).tolist()
        table, lengths, parents, shares, at = [], [], [], [0] * total, 0
        for i in range(b):
            length, shared = _group(case, i)
            each, in_common = -(-length // PAGE), shared // PAGE
            first = ids[at : at + in_common]
            at += in_common
            for p in first:
                shares[p] = n - 1
            for _ in range(n):
                rest = ids[at : at + each - in_common]
                at += each - in_common
                table.append(first + rest + [0] * (per_row - each))
            lengths += [length] * n
            found, names = _parents(case, i), torch.randperm(n, generator=order).tolist()
            parents += [-1] * n if found is None else [i * n + names[j] for j in found]
        # the list holds the pages in the order in which they were handed out; those before free_start are in use
        s.update(table=_ints(table), lengths=_ints(lengths), parents=_ints(parents), shares=_ints(shares), free=_ints(ids), free_start=_ints([at]))
        s["pools"] = [_bytes(g, total, *page_bytes) for _ in range(2 * case["layers"])]
        return s
    used, total = _compact_sizes(case)
    ids = torch.randperm(total, generator=order).tolist()
    per_row = -(-case["cache"] // PAGE) + 1
    table, lengths, at = [], [], 0
    for i in range(case["B"]):
        length = _group(case, i)[0]
        each = -(-length // PAGE)
        table.append(ids[at : at + each] + [0] * (per_row - each))
        lengths.append(length)
        at += each
    shares = (torch.randint(0, 3, (total,), generator=g, device="cuda") // 2).to(torch.int32)
    shares[torch.tensor(ids[at:], device="cuda")] = 0
    s.update(table=_ints(table), lengths=_ints(lengths), shares=shares, free=_ints(ids), free_start=_ints([at]))
    s["pools"] = [_bytes(g, total, *page_bytes) for _ in range(2 * case["layers"])]
    return s


# ---------------------------------------------------------------------------------------------- the framework's calls
def _package():
    path = os.path.abspath("tensor-product-attention-jax_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from tpa import tpa

    return tpa


def _own_run(s):
    tpa = _package()
    if s["kind"] == "select":
        return tpa.tpa_beam_select(s["logits"], s["scores"], finished=s["finished"], eos_token=EOS)
    h = s["H"]
    if s["kind"] == "write":
        tpa.tpa_cache_write_fp4(s["k"], s["v"], h, *s["pools"], s["slots"])
        return tpa.tpa_cache_read_fp4(*s["pools"], h, s["slots"][:, : s["T"]], head_dim=s["D"], dtype=s["k"].dtype)
    if s["kind"] == "decode":
        return tpa.tpa_decode_fp4(s["q"][..., :h], s["q"][..., h:], *s["pools"], sm_scale=s["D"] ** -0.5, kv_lengths=s["lengths"], page_table=s["table"],
                                  causal=tpa.CAUSAL_BOTTOM_RIGHT)
    if s["kind"] == "fork":
        out = tpa.tpa_pages_fork(s["table"], s["lengths"], s["parents"], s["shares"], s["free"], s["pools"], page_size=PAGE, free_start=s["free_start"])
    else:
        out = tpa.tpa_pages_compact(s["table"], s["lengths"], s["shares"], s["free"], s["pools"], page_size=PAGE, free_start=s["free_start"])
    return *out, *s["pools"]


# ---------------------------------------------------------------------------------------------- the plain forms
def _power_of_two(e):
    """2^e, exactly"""
    return ((e + 127).to(torch.int32) << 23).view(torch.float32)


def _plain_codes(x):
    """[..., n] values -> (codes [..., n] uint8, scales [..., ceil(n / 32)] uint8)"""
    n = x.shape[-1]
    blocks = torch.nn.functional.pad(x.float(), (0, -n % 32)).unflatten(-1, (-1, 32))
    most = blocks.abs().amax(-1)
    significand, exponent = torch.frexp(most)
    e = exponent - 3 + (significand > 7.25 / 8).to(exponent.dtype)
    e = torch.where(most == 0, -125, e).clamp(-125, 125)
    y = blocks.abs() * _power_of_two(-e)[..., None]
    y = torch.where(y < 2, (2 * y).round() / 2, torch.where(y < 4, y.round(), 2 * (y / 2).round())).clamp(max=6)
    codes = torch.where(y <= 2, 2 * y, torch.where(y <= 4, y + 2, torch.full_like(y, 7.0))).to(torch.uint8)
    codes = codes + 8 * (blocks < 0).to(torch.uint8)
    return codes.flatten(-2)[..., :n], (e + 127).to(torch.uint8)


def _plain_rows(x, h):
    """[..., h + d] factors -> rows of bytes"""
    d = x.shape[-1] - h
    (cb, sb), (ca, sa) = _plain_codes(x[..., h:]), _plain_codes(x[..., :h])
    codes = [c[..., 0::2] + 16 * c[..., 1::2] for c in (cb, ca)]
    rows = torch.cat([*codes, sb, sa], -1)
    return torch.nn.functional.pad(rows, (0, _row(h, d) - rows.shape[-1]))


def _plain_values(codes, scales):
    n = 2 * codes.shape[-1]
    of = torch.tensor(LEVELS + tuple(-x for x in LEVELS), device=codes.device)
    x = of[torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()]
    return x * _power_of_two(scales.to(torch.int32) - 127).repeat_interleave(32, -1)[..., :n]


def _plain_factors(rows, h, d):
    """rows of bytes -> (a [..., h], b [..., d]) in 32 bits"""
    at, nb = (d + h) // 2, -(-d // 32)
    b = _plain_values(rows[..., : d // 2], rows[..., at : at + nb])
    return _plain_values(rows[..., d // 2 : at], rows[..., at + nb : at + nb + -(-h // 32)]), b


def _plain_write(s):
    h, n = s["H"], s["T"]
    at = s["slots"][0, :n].long()
    out = []
    for pool, x in zip(s["pools"], (s["k"], s["v"])):
        flat = pool.view(-1, *pool.shape[2:])
        flat[at] = _plain_rows(x[0, :n], h)
        out.append(torch.cat(_plain_factors(flat[at], h, s["D"]), -1)[None].to(x.dtype))
    return tuple(out)


def _plain_decode(s):
    b, lq, h, d, rk, dtype = s["B"], s["lq"], s["H"], s["D"], s["rk"], s["q"].dtype
    keys = s["table"].shape[1] * PAGE
    q = torch.matmul(s["q"][..., :h].float().transpose(-1, -2), s["q"][..., h:].float()) * (d**-0.5 / s["rq"])
    (ka, kb), (va, vb) = (_plain_factors(p[s["table"].long()].view(b, keys, rk, -1), h, d) for p in s["pools"])
    # logits from products with the rows of the ranks, which the heads share
    of_rows = torch.matmul(q.view(b, lq * h, d), kb.view(b, keys * rk, d).transpose(1, 2).contiguous()).view(b, lq, h, keys, rk)
    x = (of_rows * ka.permute(0, 3, 1, 2)[:, None]).sum(-1) / rk
    sees = s["lengths"].long()[:, None] - lq + 1 + torch.arange(lq, device="cuda")
    x = x.masked_fill(torch.arange(keys, device="cuda") >= sees[:, :, None, None], -math.inf)
    most = x.amax(-1, keepdim=True)
    p = (x - most).exp()
    total = p.sum(-1)
    p = p / total[..., None]
    weights = (p[..., None] * va.permute(0, 3, 1, 2)[:, None]).view(b, lq * h, keys * rk)
    o = torch.matmul(weights, vb.view(b, keys * rk, d)).view(b, lq, h, d) / rk
    return o.to(dtype), (total.log() + most[..., 0]).transpose(1, 2).contiguous()


def _plain_select(s):
    b, n, vocab = s["logits"].shape
    x = s["logits"].double()  # ranks of values that lie close together
    most = x.amax(-1, keepdim=True)
    value = s["scores"].double()[..., None] + (x - most - (x - most).exp().sum(-1, keepdim=True).log())
    only = torch.full_like(value, -math.inf)
    only[..., EOS] = s["scores"].double()
    value = torch.where(s["finished"][..., None], only, value)
    value = torch.where(value.isnan(), -math.inf, value).flatten(1)
    value, at = (x[:, :n] for x in value.sort(dim=1, descending=True, stable=True))
    beam, token = at // vocab, at % vocab
    parents = beam + n * torch.arange(b, device="cuda")[:, None]
    return value.float(), parents.to(torch.int32), token.to(torch.int32), s["finished"].gather(1, beam) | (token == EOS)


def _plain_fork(s):
    table, lengths, parents = s["table"].long(), s["lengths"].long(), s["parents"].long()
    rows, per_row, total, dev = len(table), table.shape[1], len(s["shares"]), table.device
    goes_on = parents >= 0
    parent = parents.clamp(min=0)
    children = torch.zeros(rows, dtype=torch.long, device=dev).scatter_add_(0, parent, goes_on.long())
    full, tail = lengths // PAGE, lengths % PAGE
    last = table.gather(1, full.clamp(max=per_row - 1)[:, None])[:, 0]
    child = torch.arange(len(parents), device=dev)
    first = torch.full((rows,), len(parents), device=dev).scatter_reduce_(0, parent, torch.where(goes_on, child, len(parents)), "amin")
    alone = s["shares"].long()[last] == 0
    keeps = (tail > 0) & (children > 0) & alone  # the first child has the parent's last page
    copies = goes_on & (tail[parent] > 0) & ~(alone[parent] & (first[parent] == child))
    start = s["free_start"].long()
    nth = start + copies.cumsum(0) - 1
    has_page = copies & (nth < len(s["free"]))
    taken = has_page.sum()
    fresh = s["free"].long()[nth.clamp(0, len(s["free"]) - 1)]
    length = torch.where(goes_on, torch.where(copies & ~has_page, full[parent] * PAGE, lengths[parent]), 0)
    entry = torch.arange(per_row, device=dev)
    new = torch.where(entry < ((length + PAGE - 1) // PAGE)[:, None], table[parent], 0)
    new = torch.where(has_page[:, None] & (entry == full[parent][:, None]), fresh[:, None], new)
    # holders of the pages
    change = torch.where(entry < full[:, None], children[:, None] - 1, 0)
    change = torch.where((entry == full[:, None]) & (tail > 0)[:, None], keeps.long()[:, None] - 1, change)
    shares = s["shares"].long().scatter_add(0, table.flatten(), change.flatten())
    released = shares < 0
    place = start + taken - released.sum() + released.cumsum(0) - 1
    free = torch.cat([s["free"], s["free"][:1]])
    free[torch.where(released & (place >= 0), place, len(free) - 1)] = torch.arange(total, device=dev, dtype=torch.int32)
    src, dst = torch.where(has_page, last[parent], table[0, 0]), torch.where(has_page, fresh, table[0, 0])  # the others write a page in use as it is
    for pool in s["pools"]:
        filled = torch.arange(PAGE, device=dev) < torch.where(has_page, tail[parent], 0)[:, None]
        pool[dst] = torch.where(filled[:, :, None, None], pool[src], pool[dst])
    to = torch.int32
    return new.to(to), length.to(to), shares.clamp(min=0).to(to), free[:-1], (start + taken - released.sum()).clamp(min=0).to(to)


def _plain_compact(s):
    total, dev = len(s["shares"]), s["table"].device
    listed_at = torch.arange(len(s["free"]), device=dev)
    is_free = torch.zeros(total + 1, dtype=torch.bool, device=dev)
    is_free[torch.where(listed_at >= s["free_start"], s["free"].long(), total)] = True
    is_free = is_free[:-1]
    page = torch.arange(total, device=dev)
    n_free = int(is_free.sum())
    n_used = total - n_free
    holes, movers = page[is_free & (page < n_used)], page[~is_free & (page >= n_used)]
    moved = page.clone()
    moved[movers] = holes
    for pool in s["pools"]:
        pool[holes] = pool[movers]
    shares = torch.zeros_like(s["shares"])
    shares[moved[~is_free]] = s["shares"][~is_free]
    free = s["free"].clone()
    free[len(free) - n_free :] = page[n_used:].to(torch.int32)
    used = torch.arange(s["table"].shape[1], device=dev) < ((s["lengths"] + PAGE - 1) // PAGE)[:, None]
    table = torch.where(used, moved[s["table"].long()], 0)
    start = torch.full((1,), len(free) - n_free, dtype=torch.int32, device=dev)
    return table.to(torch.int32), shares, free, start, moved.to(torch.int32)


def run(state):
    if own:
        return _own_run(state)
    kind = state["kind"]
    if kind == "write":
        return _plain_write(state)
    if kind == "decode":
        return _plain_decode(state)
    if kind == "select":
        return _plain_select(state)
    return *(_plain_fork if kind == "fork" else _plain_compact)(state), *state["pools"]


# ---------------------------------------------------------------------------------------------- from the definitions, in 64 bits
def exact(case, seed):
    if case["kind"] in ("fork", "compact"):
        return None  # whole numbers
    s = prepare(case, seed)
    if case["kind"] == "select":
        return _exact_select(s)
    h, d = case["H"], case["D"]
    if case["kind"] == "write":
        return tuple(torch.cat([_exact_held(x[0, : case["T"], :, :h].double()), _exact_held(x[0, : case["T"], :, h:].double())], -1)[None] for x in (s["k"], s["v"]))
    return _exact_decode(s, h, d)


def _exact_held(x):
    """What 4 bits and a scale hold of x: the nearest level of each block of 32, an even code where two are as near."""
    levels = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)
    halfway = (levels[1:] + levels[:-1]) / 2
    out = torch.empty_like(x)
    for first in range(0, x.shape[-1], 32):
        block = x[..., first : first + 32]
        most = block.abs().amax(-1, keepdim=True)
        e = torch.floor(torch.log2(most)) - 2
        step = torch.pow(2.0, torch.where(most > 7.25 * torch.pow(2.0, e), e + 1, e).clamp(-125, 125))
        size = block.abs() / step
        code = sum(((size >= at) if i % 2 else (size > at)).long() for i, at in enumerate(halfway.tolist()))
        out[..., first : first + 32] = torch.sign(block) * levels[code] * step
    return out


def _exact_select(s):
    b, n, vocab = s["logits"].shape
    best = torch.empty((b, n), dtype=torch.float64, device="cuda")
    for i in range(b):
        value = torch.log_softmax(s["logits"][i].double(), -1) + s["scores"][i].double()[:, None]
        for j in torch.nonzero(s["finished"][i])[:, 0].tolist():
            value[j] = -math.inf
            value[j, EOS] = s["scores"][i, j].double()
        best[i] = torch.topk(value.flatten(), n).values
    return best, None, None, None


def _exact_decode(s, h, d):
    lq, rk = s["lq"], s["rk"]
    o = torch.empty((s["B"], lq, h, d), dtype=torch.float64, device="cuda")
    lse = torch.empty((s["B"], h, lq), dtype=torch.float64, device="cuda")
    level = torch.tensor([(-1) ** (c // 8) * LEVELS[c % 8] for c in range(16)], dtype=torch.float64, device="cuda")

    def values(rows, first, count, scales):
        at = torch.arange(count, device="cuda")
        codes = (rows[..., first + at // 2].long() >> (4 * (at % 2))) % 16
        return level[codes] * torch.pow(2.0, rows[..., scales + at // 32].double() - 127)

    def heads(rows):  # [tokens, rk, bytes] -> [h, tokens, d]
        b, a = values(rows, 0, d, (d + h) // 2), values(rows, d // 2, h, (d + h) // 2 + -(-d // 32))
        return sum(a[:, r, :, None] * b[:, r, None] for r in range(rk)).transpose(0, 1) / rk

    for i, length in enumerate(s["lengths"].tolist()):
        t = torch.arange(length, device="cuda")
        at = s["table"][i].long()[t // PAGE]
        k, v = (heads(p[at, t % PAGE]) for p in s["pools"])
        x = s["q"][i].double()
        q = sum(x[:, r, :h, None] * x[:, r, None, h:] for r in range(s["rq"])).transpose(0, 1) / s["rq"] / math.sqrt(d)
        logits = q @ k.transpose(1, 2).contiguous()
        logits[:, t > (length - lq + torch.arange(lq, device="cuda"))[:, None]] = -math.inf
        lse[i] = torch.logsumexp(logits, -1)
        o[i] = (torch.softmax(logits, -1) @ v).transpose(0, 1)
    return o, lse
