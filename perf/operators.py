"""The operators of a serving step over a cache held in 8 bits, in plain torch and as calls of the framework.

`plan`: from the tokens that requests hold and bring, on the GPU, the index arrays of a step, slots in the pool and the growth of the block
table. `append`: new rows into a cache whose blocks of 16 tokens share a scale per kv head (K and V apart), and the blocks they went to read
back. `attend`: attention over such a cache, one query per sequence or ragged causal chunks.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 16  # tokens that share a scale
TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
ELEM = {"bf16": 2, "f16": 2, "f32": 4}
MOST = {"i8": 127.0, "f8": 448.0}  # largest value of a code
FLOOR = 2.0 ** -100  # smallest scale


def listed():
    return [
        # a full server decoding: every request brings one token, a sixteenth of them need a page
        dict(name="plan_decode", op="plan", seqs=64, low=1, high=4096, short=1, long=1, page=16),
        # an iteration of continuous batching: pieces of prompts beside decoding requests, some sitting the step out
        dict(name="plan_mixed", op="plan", seqs=300, low=0, high=3000, short=0, long=140, page=16),
        # a batch job's prompts, laid out at once
        dict(name="plan_prompts", op="plan", seqs=4000, low=0, high=700, short=1, long=512, page=32),
        # a token of each of 64 conversations
        dict(name="append_step", op="append", seqs=64, low=1, high=4096, short=1, long=1, heads=12, kv_heads=2, dim=128, dtype="bf16", store="i8",
             page=16),
        # pieces of prompts that begin and end inside blocks
        dict(name="append_pieces", op="append", seqs=24, low=1, high=3000, short=1, long=200, heads=32, kv_heads=8, dim=64, dtype="f16",
             store="f8", page=32),
        # sixteen whole prompts
        dict(name="append_prompts", op="append", seqs=16, low=0, high=0, short=4096, long=4096, heads=12, kv_heads=2, dim=128, dtype="bf16",
             store="i8", page=16),
        # one user in the middle of a short answer
        dict(name="decode_one", op="attend", seqs=1, low=776, high=776, short=1, long=1, heads=12, kv_heads=2, dim=128, dtype="bf16", store="i8",
             page=16, window=0, keep=0),
        # a full server's step: 64 conversations of 4096 tokens
        dict(name="decode_batch", op="attend", seqs=64, low=4095, high=4095, short=1, long=1, heads=12, kv_heads=2, dim=128, dtype="bf16",
             store="i8", page=16, window=0, keep=0),
        # ragged conversations of a model in 32 bits with a window that keeps the first tokens
        dict(name="decode_window", op="attend", seqs=24, low=100, high=9000, short=1, long=1, heads=32, kv_heads=8, dim=64, dtype="f32",
             store="f8", page=32, window=2000, keep=4),
        # chunked prefill of eight conversations
        dict(name="chunk_serving", op="attend", seqs=8, low=0, high=8192, short=512, long=512, heads=12, kv_heads=2, dim=128, dtype="bf16",
             store="i8", page=16, window=0, keep=0),
        # a whole prompt at once
        dict(name="chunk_prompt", op="attend", seqs=1, low=0, high=0, short=5000, long=5000, heads=32, kv_heads=8, dim=128, dtype="f16",
             store="f8", page=16, window=0, keep=0),
        # decode rows and small pieces of prompts side by side, with a window
        dict(name="chunk_mixed", op="attend", seqs=24, low=1, high=3000, short=1, long=96, heads=32, kv_heads=8, dim=64, dtype="f16", store="i8",
             page=32, window=1000, keep=0),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _drawn(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "attend"])
    page = rng.choice([16, 16, 32, 64])
    if op == "plan":
        seqs = _log(rng, 1, 4000)
        long = max(1, _log(rng, 1, 900000) // seqs)
        return dict(op=op, seqs=seqs, low=rng.randint(0, 500), high=rng.randint(500, 6000), short=rng.randint(0, long), long=long, page=page)
    kv_heads = rng.choice([1, 2, 2, 4, 8])
    shape = dict(heads=kv_heads * rng.choice([1, 4, 4, 6, 6, 8, 16]), kv_heads=kv_heads, dim=rng.choice([64, 128, 128, 128, 256]),
                 dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), store=rng.choice(["i8", "i8", "f8"]), page=page)
    if op == "append":
        seqs = _log(rng, 1, 64)
        long = max(1, _log(rng, 1, 65536) // seqs)
        high = _log(rng, 1, 4096)
        return dict(op=op, seqs=seqs, low=rng.randint(0, high), high=high, short=rng.randint(1, long), long=long, **shape)
    seqs = _log(rng, 1, 64)
    single = rng.random() < 0.5
    long = 1 if single else max(2, _log(rng, 2, 5000) // seqs)
    high = max(1, _log(rng, 16, 65536 if single else 8192) // (seqs if single and seqs > 8 else 1))
    window = rng.choice([0, 0, 0, _log(rng, 16, 4096)])
    return dict(op=op, seqs=seqs, low=rng.randint(0, high), high=high, short=1 if single else rng.randint(1, long), long=long, window=window,
                keep=rng.choice([0, 4, 20]) if window else 0, **shape)


def _too_much(case):
    """Whether a case costs more than the largest listed one, by its work or in its plain form's memory."""
    if case["op"] == "plan":
        return False
    held, new = _sizes(case)
    longest = int((held + new).max())
    cells = case["seqs"] * longest * case["kv_heads"] * case["dim"]
    if cells > 64 * 4096 * 2 * 128:
        return True
    if case["op"] == "append":
        return False
    return case["seqs"] * case["heads"] * int(new.max()) * longest > 32 * 5000 * 5000 or work(case)["flops"] > 2e11


def draw(rng):
    while True:
        case = _drawn(rng)
        if not _too_much(case):
            return case


# ---- sizes ---------------------------------------------------------------------------------------------------------------


def _sizes(case):
    """Tokens held and brought, of every sequence: of the case alone, so that its work does not depend on a seed."""
    rng = np.random.default_rng([int(case[k]) for k in ("seqs", "low", "high", "short", "long")])
    held = rng.integers(case["low"], case["high"] + 1, case["seqs"])
    return held, rng.integers(case["short"], case["long"] + 1, case["seqs"])


def _visible(case, held, new):
    """Keys that all queries of a sequence see together, and the tokens that any of them sees."""
    pairs = tokens = 0
    window, keep = case["window"], case["keep"]
    for h, n in zip(held.tolist(), new.tolist()):
        at = np.arange(h, h + n, dtype=np.int64)  # positions of the queries
        if window == 0:
            pairs += int((at + 1).sum())
            tokens += h + n
        else:
            first = np.maximum(at + 1 - window, 0)
            pairs += int((at + 1 - first + np.minimum(first, keep)).sum())
            tokens += h + n - int(first[0]) + min(keep, int(first[0]))
    return pairs, tokens


def work(case):
    held, new = _sizes(case)
    rows = int(new.sum())
    if case["op"] == "plan":
        grown = int((-(-(held + new) // case["page"]) + -held // case["page"]).sum())
        return {"bytes": 8 * case["seqs"] + 12 * case["seqs"] + 16 * rows + 8 * grown, "flops": 0}
    kv_heads, dim, elem = case["kv_heads"], case["dim"], ELEM[case["dtype"]]
    if case["op"] == "append":
        back = int((held % BLOCK + new).sum())  # tokens of the blocks that were written to
        blocks = int((-(-(held % BLOCK + new) // BLOCK)).sum())
        return {"bytes": 2 * kv_heads * (dim * (elem + 1) * (rows + back) + 8 * blocks) + 8 * (rows + back), "flops": 0}
    pairs, tokens = _visible(case, held, new)
    return {"bytes": kv_heads * tokens * (2 * dim + 8 / BLOCK) + 2 * rows * case["heads"] * dim * elem, "flops": 4 * dim * case["heads"] * pairs}


# ---- inputs --------------------------------------------------------------------------------------------------------------


def _i32(values):
    return torch.from_numpy(np.ascontiguousarray(values, dtype=np.int32)).cuda()


def _rows_of(held, new):
    """Sequence and position of every new row, sequences back to back."""
    seq = np.repeat(np.arange(len(new)), new)
    return seq, np.arange(len(seq)) - np.repeat(np.cumsum(new) - new, new) + np.repeat(held, new)


def _values(case, gen, *shape):
    """Rows of a head's keys or values: heads of different size and a few channels that stand out, as projections give them."""
    x = torch.randn(*shape, generator=gen, device="cuda")
    x *= 0.5 + torch.rand(shape[-2], 1, generator=gen, device="cuda")
    x *= torch.where(torch.rand(shape[-2], shape[-1], generator=gen, device="cuda") < 0.02, 6.0, 1.0)
    return x.to(TORCH[case["dtype"]])


def _tables(case, held, new, rng):
    """Pages of every sequence for all its tokens, in the order of a pool that has been used."""
    counts = -(-(held + new) // case["page"])
    order = rng.permutation(int(counts.sum()))
    table = np.zeros((len(counts), max(1, int(counts.max()))), dtype=np.int32)
    at = 0
    for i, n in enumerate(counts.tolist()):
        table[i, :n] = order[at:at + n]
        at += n
    return table, len(order)


class _Pool:
    """The plain form's cache: codes [page, K | V, kv head, slot, dim] and a scale for every block of 16 slots and head."""

    def __init__(self, case, pages):
        blocks = case["page"] // BLOCK
        kind = torch.int8 if case["store"] == "i8" else torch.float8_e4m3fn
        self.codes = torch.zeros(pages * blocks, 2, case["kv_heads"], BLOCK, case["dim"], dtype=torch.int8, device="cuda").view(kind)
        self.scales = torch.zeros(pages * blocks, 2, case["kv_heads"], device="cuda")


def _framework_cache(case, table, pages):
    import llaisys_b200 as llaisys

    cache = llaisys.PagedKVCache.quantized(
        pages, case["kv_heads"], case["dim"], store=llaisys.DataType.I8 if case["store"] == "i8" else llaisys.DataType.F8,
        dtype={"bf16": llaisys.DataType.BF16, "f16": llaisys.DataType.F16, "f32": llaisys.DataType.F32}[case["dtype"]],
        page_size=case["page"], device=llaisys.DeviceType.NVIDIA, max_seqs=len(table), max_pages_per_seq=table.shape[1])
    held, new = _sizes(case)
    for row, n in zip(table, (-(-(held + new) // case["page"])).tolist()):
        cache.assign_pages(cache.add_seq(), row[:n])
    cache.flush()
    return cache


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _append(state, k, v, seq, pos):
    """New rows into the cache of a state, in either form."""
    if own:
        state["cache"].append_dev(0, k, v, seq, pos, len(seq), _stream())
    else:
        _plain_append(state, k, v, seq, pos)


def prepare(case, seed):
    gen, rng = torch.Generator(device="cuda").manual_seed(seed), np.random.default_rng(seed)
    held, new = _sizes(case)
    if case["op"] == "plan":
        return _prepare_plan(case, held, new, rng)
    table, pages = _tables(case, held, new, rng)
    state = dict(case=case, table=_i32(table), pool=None if own else _Pool(case, pages), cache=_framework_cache(case, table, pages) if own else None)
    kv_heads, dim = case["kv_heads"], case["dim"]

    def rows(before, count):
        seq, pos = _rows_of(before, count)
        n = len(seq)
        return _values(case, gen, n, kv_heads, dim), _values(case, gen, n, kv_heads, dim), _i32(seq), _i32(pos)

    if held.sum():
        _append(state, *rows(np.zeros_like(held), held))  # what the sequences hold
    state["new"] = rows(held, new)
    seqs, nh = case["seqs"], case["heads"]
    state["lens"], state["starts"] = _i32(held + new), _i32(np.concatenate([[0], np.cumsum(new)]))
    n = int(new.sum())
    if case["op"] == "append":  # the tokens of every block that the rows go to
        seq, pos = _rows_of(held // BLOCK * BLOCK, held % BLOCK + new)
        state["back"] = (_i32(seq), _i32(pos))
        state["out"] = [torch.empty(len(seq), kv_heads, dim, dtype=TORCH[case["dtype"]], device="cuda") for _ in range(2)] if own else None
        return state
    _append(state, *state["new"])
    del state["new"]
    state |= dict(q=torch.randn(n, nh, dim, generator=gen, device="cuda").to(TORCH[case["dtype"]]), ids=_i32(np.arange(seqs)), rows=n,
                  longest=int((held + new).max()), most=int(new.max()),
                  out=torch.empty(n, nh, dim, dtype=TORCH[case["dtype"]], device="cuda") if own else None)
    return state


def _prepare_plan(case, held, new, rng):
    page, seqs = case["page"], case["seqs"]
    before, after = -(-held // page), -(-(held + new) // page)
    stride, used, grown = max(1, int(after.max())), int(before.sum()), int((after - before).sum())
    pages = rng.permutation(used + grown + 100)
    table = np.full((seqs + 5, stride), -1, dtype=np.int32)  # the batch's requests have some of the server's rows
    ids = rng.permutation(seqs + 5)[:seqs]
    at = 0
    for i, n in zip(ids.tolist(), before.tolist()):
        table[i, :n] = pages[at:at + n]
        at += n
    rows = -(-int(new.sum()) // 64) * 64 + 64  # as a program rounds it up that replays its step as a graph
    state = dict(case=case, ids=_i32(ids), held=_i32(held), new=_i32(new), free=_i32(pages[used:]), table=_i32(table), rows=rows)
    if own:
        state["out"] = dict(q_starts=torch.empty(seqs + 1, dtype=torch.int32, device="cuda"),
                            kv_lens=torch.empty(seqs, dtype=torch.int32, device="cuda"),
                            page_starts=torch.empty(seqs + 1, dtype=torch.int32, device="cuda"),
                            row_seqs=torch.empty(rows, dtype=torch.int32, device="cuda"),
                            row_positions=torch.empty(rows, dtype=torch.int32, device="cuda"),
                            row_slots=torch.empty(rows, dtype=torch.int64, device="cuda"),
                            status=torch.empty(2, dtype=torch.int32, device="cuda"))
    return state


# ---- the operators -------------------------------------------------------------------------------------------------------


def run(state):
    op = state["case"]["op"]
    if op == "plan":
        return _own_plan(state) if own else _plain_plan(state)
    if op == "append":
        _append(state, *state["new"])
        if not own:
            return _plain_back(state)
        seq, pos = state["back"]
        state["cache"].gather_dev(0, state["out"][0], state["out"][1], seq, pos, len(seq), _stream())
        return state["out"]
    return _own_attend(state) if own else _plain_attend(state)


def _own_plan(state):
    import llaisys_b200 as llaisys

    out, table = state["out"], state["table"]
    llaisys.paged_plan_dev(
        stream=_stream(), seq_ids_dev=state["ids"], held_dev=state["held"], new_dev=state["new"], n_seqs=len(state["ids"]),
        page_size=state["case"]["page"], n_rows=state["rows"], free_pages_dev=state["free"], n_free=len(state["free"]), block_table_dev=table,
        table_rows=table.shape[0], table_stride=table.shape[1], q_starts_dev=out["q_starts"], kv_lens_dev=out["kv_lens"],
        page_starts_dev=out["page_starts"], row_seqs_dev=out["row_seqs"], row_positions_dev=out["row_positions"],
        row_slots_dev=out["row_slots"], status_dev=out["status"])
    return dict(out, table=table)


def _own_attend(state):
    case, cache, out = state["case"], state["cache"], state["out"]
    scale = 1 / math.sqrt(case["dim"])
    starts = None if case["long"] == 1 else state["starts"]
    if case["window"]:
        cache.attention_dev(0, out, state["q"], state["ids"], starts, state["lens"], n_seqs=case["seqs"], total_q=state["rows"],
                            max_q_len=state["most"], max_kv_len=state["longest"], nh=case["heads"], scale=scale, stream=_stream(),
                            window=case["window"], keep_first=case["keep"])
    elif starts is None:
        cache.decode_dev(0, out, state["q"], state["ids"], state["lens"], case["seqs"], state["longest"], case["heads"], scale, _stream())
    else:
        cache.prefill_dev(0, out, state["q"], state["ids"], starts, state["lens"], case["seqs"], state["rows"], state["most"], state["longest"],
                          case["heads"], scale, _stream())
    return out


def _starts(counts):
    """Exclusive prefix sums with the total at the end."""
    return torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), torch.cumsum(counts, 0)])


def _plain_plan(state):
    page, ids, table = state["case"]["page"], state["ids"].long(), state["table"]
    held, new = state["held"].long(), state["new"].long()
    kv = held + new
    q_starts, before, after = _starts(new), (held + page - 1) // page, (kv + page - 1) // page
    grown = _starts(after - before)
    # growth: entry j of the free list goes to the request whose range holds it
    j = torch.arange(len(state["free"]), device="cuda")
    owner = torch.searchsorted(grown, j, right=True) - 1
    taken = j < grown[-1]
    owner = torch.where(taken, owner, 0)
    at = torch.where(taken, ids[owner] * table.shape[1] + before[owner] + j - grown[owner], table.numel())
    table.copy_(torch.cat([table.view(-1), table.view(-1)[:1]]).scatter_(0, at, state["free"])[:-1].view(table.shape))
    # rows
    r = torch.arange(state["rows"], device="cuda")
    seq = torch.searchsorted(q_starts, r, right=True) - 1
    live = r < q_starts[-1]
    seq = torch.where(live, seq, 0)
    pos = held[seq] + r - q_starts[seq]
    entry = table[ids[seq], torch.where(live, pos // page, 0)].long()
    slots = entry * page + pos % page
    status = torch.stack([grown[-1], torch.zeros_like(grown[-1])])
    return dict(q_starts=q_starts.int(), kv_lens=kv.int(), page_starts=_starts(after).int(), row_seqs=torch.where(live, ids[seq], -1).int(),
                row_positions=torch.where(live, pos, -1).int(), row_slots=torch.where(live, slots, -1), status=status.int(), table=table)


def _code(x, store):
    """Codes of numbers that are already divided by their scale."""
    if store == "i8":
        return torch.clamp(torch.round(x), -127, 127).to(torch.int8)
    return torch.clamp(x, -448, 448).to(torch.float8_e4m3fn)


def _plain_append(state, k, v, seq, pos):
    case, pool = state["case"], state["pool"]
    store, most, blocks_per_page = case["store"], MOST[case["store"]], case["page"] // BLOCK
    seq, pos = seq.long(), pos.long()
    block = state["table"][seq, pos // case["page"]].long() * blocks_per_page + pos % case["page"] // BLOCK
    rows = torch.stack([k, v], 1).float()  # [rows, 2, kv head, dim]
    touched, index = torch.unique(block, return_inverse=True)
    largest = torch.zeros(len(touched), 2, case["kv_heads"], device="cuda")
    largest.scatter_reduce_(0, index[:, None, None].expand(-1, 2, case["kv_heads"]), rows.abs().amax(-1), "amax")
    first = torch.full((len(touched),), BLOCK, device="cuda").scatter_reduce_(0, index, pos % BLOCK, "amin")
    old = torch.where((first > 0)[:, None, None], pool.scales[touched], 0.0)
    scale = torch.maximum(old, largest / torch.full_like(largest, most)).clamp_min(FLOOR)  # (a division by a plain number would be a product)
    inverse = 1.0 / scale
    # what the block held in front of the new rows, in the new scale
    codes = pool.codes[touched]
    again = (scale > old)[:, :, :, None, None] & (torch.arange(BLOCK, device="cuda") < first[:, None])[:, None, None, :, None]
    factor = (old * inverse)[..., None, None]
    pool.codes[touched] = torch.where(again, _code(codes.float() * factor, store).view(torch.int8), codes.view(torch.int8)).view(codes.dtype)
    pool.scales[touched] = scale
    pool.codes.view(torch.int8)[block, :, :, pos % BLOCK] = _code(rows * inverse[index][..., None], store).view(torch.int8)


def _plain_back(state):
    case, pool = state["case"], state["pool"]
    seq, pos = (x.long() for x in state["back"])
    block = state["table"][seq, pos // case["page"]].long() * (case["page"] // BLOCK) + pos % case["page"] // BLOCK
    rows = pool.codes.view(torch.int8)[block, :, :, pos % BLOCK].view(pool.codes.dtype).float() * pool.scales[block][..., None]
    rows = rows.to(TORCH[case["dtype"]])
    return [rows[:, 0], rows[:, 1]]


def _plain_attend(state):
    case, pool = state["case"], state["pool"]
    seqs, kv_heads, dim, nh = case["seqs"], case["kv_heads"], case["dim"], case["heads"]
    longest, most, group = state["longest"], state["most"], nh // kv_heads
    lens, starts = state["lens"].long(), state["starts"].long()
    counts = starts[1:] - starts[:-1]
    # keys and values of all sequences side by side, [seq, K | V, kv head, token, dim]
    blocks = -(-longest // BLOCK)
    b = torch.arange(blocks, device="cuda") * BLOCK
    at = state["table"][:, b // case["page"]].long() * (case["page"] // BLOCK) + b % case["page"] // BLOCK
    kv = pool.codes.view(torch.int8)[at].view(pool.codes.dtype).float() * pool.scales[at][..., None, None]
    kv = kv.permute(0, 2, 3, 1, 4, 5).reshape(seqs, 2, kv_heads, blocks * BLOCK, dim)[:, :, :, :longest]
    # queries, [seq, kv head, query x head of the group, dim]
    r = torch.arange(state["rows"], device="cuda")
    seq = torch.searchsorted(starts, r, right=True) - 1
    t = r - starts[seq]
    q = torch.zeros(seqs, most, nh, dim, device="cuda")
    q[seq, t] = state["q"].float()
    q = q.view(seqs, most, kv_heads, group, dim).transpose(1, 2).reshape(seqs, kv_heads, most * group, dim)
    score = torch.matmul(q, kv[:, 0].transpose(-1, -2)).view(seqs, kv_heads, most, group, longest) * (1 / math.sqrt(dim))
    i = (lens - counts)[:, None, None] + torch.arange(most, device="cuda")[:, None]
    j = torch.arange(longest, device="cuda")
    seen = (j <= i) & (j < lens[:, None, None])
    if case["window"]:
        seen &= (i - j < case["window"]) | (j < case["keep"])
    score.masked_fill_(~seen[:, None, :, None], -math.inf)
    score -= score.amax(-1, keepdim=True).clamp_min(-1e30)
    weight = score.exp_()
    weight /= weight.sum(-1, keepdim=True).clamp_min(1e-30)
    out = torch.matmul(weight.view(seqs, kv_heads, most * group, longest), kv[:, 1])
    out = out.view(seqs, kv_heads, most, group, dim).transpose(1, 2).reshape(seqs, most, nh, dim)
    return out[seq, t].to(TORCH[case["dtype"]])


# ---- the same from the definitions, in 64 bits ---------------------------------------------------------------------------


def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    gen, rng = torch.Generator(device="cuda").manual_seed(seed), np.random.default_rng(seed)
    held, new = _sizes(case)
    _tables(case, held, new, rng)
    shape = (case["kv_heads"], case["dim"])
    parts = []
    for count in (held, new):
        n = int(count.sum())
        if n or count is new:
            parts.append([list(torch.split(_values(case, gen, n, *shape).double(), count.tolist())) for _ in range(2)])
        else:
            parts.append([[torch.zeros(0, *shape, dtype=torch.float64, device="cuda") for _ in count] for _ in range(2)])
    if case["op"] == "append":
        return [torch.cat([_exact_rows(case, a, b)[int(h) // BLOCK * BLOCK:] for h, a, b in zip(held, parts[0][kv], parts[1][kv])])
                for kv in (0, 1)]
    nh, dim, group = case["heads"], case["dim"], case["heads"] // case["kv_heads"]
    q = torch.randn(int(new.sum()), nh, dim, generator=gen, device="cuda").to(TORCH[case["dtype"]]).double()
    out, row = torch.zeros_like(q), 0
    for s in range(case["seqs"]):
        k, v = (_exact_rows(case, parts[0][kv][s], parts[1][kv][s]) for kv in (0, 1))
        i = torch.arange(int(held[s]), int(held[s] + new[s]), device="cuda")[:, None]
        j = torch.arange(len(k), device="cuda")[None, :]
        hidden = j > i
        if case["window"]:
            hidden |= (i - j >= case["window"]) & (j >= case["keep"])
        for h in range(nh):
            x = (q[row:row + len(i), h] @ k[:, h // group].T / math.sqrt(dim)).masked_fill(hidden, -math.inf)
            out[row:row + len(i), h] = torch.softmax(x, -1) @ v[:, h // group]
        row += len(i)
    return out


def _exact_rows(case, held, new):
    """What a sequence's rows are worth after `held` and then `new` were appended. A scale, its inverse and the factor between two scales are
    numbers of 32 bits by definition; everything else is in 64."""
    most = MOST[case["store"]]

    def single(x):
        return x.float().double()

    def code(x):
        if case["store"] == "i8":
            return torch.round(single(x))
        x = single(x)
        step = 2.0 ** (torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
        return torch.round(x / step).mul(step).clamp(-448, 448)

    def blocks(x):
        pad = -len(x) % BLOCK
        return torch.cat([x, x.new_zeros(pad, *x.shape[1:])]).view(-1, BLOCK, *x.shape[1:])

    def scale_of(b, least):
        return torch.maximum(torch.maximum(single(b.abs().amax((1, 3)) / most), least), torch.full_like(least, FLOOR))

    shape = new.shape[1:]
    none = torch.zeros(1, shape[0], dtype=torch.float64, device="cuda")
    h = blocks(held)
    s = scale_of(h, none) if len(h) else none[:0]
    c = code(h * single(1 / s)[:, None, :, None])
    rest = len(held) % BLOCK
    whole = len(held) // BLOCK
    # the block that `new` begins in
    head = new[:BLOCK - rest] if rest else new[:0]
    if len(head):
        old = s[whole:]
        grown = scale_of(head[None], old)
        factor = single(old * single(1 / grown))
        kept = torch.where((grown > old)[:, None, :, None], code(c[whole:, :rest] * factor[:, None, :, None]), c[whole:, :rest])
        joined = torch.cat([kept[0], code(head * single(1 / grown)[0][:, None])])
        c, s = torch.cat([c[:whole], blocks(joined)]), torch.cat([s[:whole], grown])
    tail = blocks(new[len(head):])
    if len(tail):
        t = scale_of(tail, none)
        c, s = torch.cat([c, code(tail * single(1 / t)[:, None, :, None])]), torch.cat([s, t])
    return (c * s[:, None, :, None]).reshape(-1, *shape)[:len(held) + len(new)]
