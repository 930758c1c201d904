"""A paged cache held in 8 bits: append, rows read back and attention against the definitions, refusals, and a step planned on the GPU.

The reference of the append is the definition in numpy, in f32 where the definition says so: rows read back have to equal it. Attention is
compared with softmax in float64 over what the cache is worth.
"""
import ctypes

import numpy as np
import pytest
import torch

import llaisys_b200 as llaisys
from llaisys_b200.libllaisys import LIB_LLAISYS, LlaisysPagedPlan, Status

BLOCK = 16
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
NAMES = {"f32": llaisys.DataType.F32, "f16": llaisys.DataType.F16, "bf16": llaisys.DataType.BF16}
STORES = {"i8": llaisys.DataType.I8, "f8": llaisys.DataType.F8}
MOST = {"i8": np.float32(127), "f8": np.float32(448)}


# ---- the definitions -----------------------------------------------------------------------------------------------------


def code(x, store):
    """Nearest code of f32 numbers that are divided by their scale, as the f32 number that it is."""
    if store == "i8":
        return np.clip(np.rint(x), -127, 127).astype(np.float32)
    return torch.from_numpy(np.clip(x, -448, 448)).to(torch.float8_e4m3fn).float().numpy()


class Definition:
    """K (or V) of one sequence: codes [token, head, dim] and a scale per block and head."""

    def __init__(self, nkvh, d, store):
        self.store, self.nkvh, self.d = store, nkvh, d
        self.codes = np.zeros((0, nkvh, d), np.float32)
        self.scales = np.zeros((0, nkvh), np.float32)

    def append(self, at, rows):  # rows f32 [n, head, dim] to tokens at, at + 1, ...
        n = at + len(rows)
        if n > len(self.codes):
            self.codes = np.concatenate([self.codes, np.zeros((n - len(self.codes), self.nkvh, self.d), np.float32)])
            blocks = -(-n // BLOCK)
            self.scales = np.concatenate([self.scales, np.zeros((max(0, blocks - len(self.scales)), self.nkvh), np.float32)])
        while len(rows):
            b, slot = divmod(at, BLOCK)
            part, rows = rows[:BLOCK - slot], rows[BLOCK - slot:]
            for h in range(self.nkvh):
                x = part[:, h]
                old = self.scales[b, h] if slot else np.float32(0)
                if not np.isfinite(x).all() or np.isnan(old):
                    self.scales[b, h] = np.nan
                    self.codes[at:at + len(part), h] = 0
                    continue
                new = np.maximum(np.maximum(old, np.abs(x).max() / MOST[self.store]), np.float32(2.0 ** -100))
                inverse = np.float32(1) / new
                if new > old and slot:
                    front = self.codes[b * BLOCK:at, h]
                    self.codes[b * BLOCK:at, h] = code(front * (old * inverse), self.store)
                self.codes[at:at + len(part), h] = code(x * inverse, self.store)
                self.scales[b, h] = new
            at += len(part)

    def worth(self):  # f32, products rounded once
        return self.codes * np.repeat(self.scales, BLOCK, 0)[:len(self.codes), :, None]


def attention_f64(q, k, v, held, scale, window=0, keep=0):
    """q [n, nh, d], k / v [tokens, nkvh, d] float64; query t sits at position held + t. -> output, and for every (row, head) the error that a
    weight or a score may bring: max |v| and max sum |q| |k|."""
    n, nh, d = q.shape
    group = nh // k.shape[1]
    i, j = torch.arange(n)[:, None] + held, torch.arange(len(k))[None, :]
    seen = j <= i
    if window:
        seen &= (i - j < window) | (j < keep)
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    s = torch.einsum("thd,jhd->htj", q, k) * scale
    s = s.masked_fill(~seen, -torch.inf)
    p = torch.where(seen.any(-1)[None, :, None], torch.softmax(s, -1), 0.0)
    big = (torch.einsum("thd,jhd->htj", q.abs(), k.abs()) * abs(scale)).masked_fill(~seen, 0).amax(-1).T
    top = torch.where(seen[None], v.abs().amax(-1).T[:, None, :], 0).amax(-1).T
    return torch.einsum("htj,jhd->thd", p, v), top, big


def tolerance(want, top, big, dtype, tokens, d):
    """Half a step of the output's type, and for the arithmetic in between: scores are f32 sums of d / 16 partial sums of exact products (each
    addition off by 2^-23 of the sum of magnitudes, by cutting), the query is carried to 2^-22 and factors cost 4 roundings; a score off by e
    moves the output by 2 e max |v|. Weights are rounded to 16 bits for 16-bit types (2^-11 relative, weights below 2^-28 of the largest to 2^-39)
    and carried to 2^-21 for f32; sums over the tokens add 2^-23 per 16 of them."""
    half = torch.finfo(TORCH[dtype]).eps / 2
    score = (d / 16 + 8) * 2.0 ** -22 * big
    weight = (2.0 ** -21 if dtype == "f32" else 2.0 ** -11 * 1.01) + (tokens / 16 + 16) * 2.0 ** -23
    return half * want.abs() + ((2 * score + 2 * weight) * top)[..., None] + 1e-30


# ---- calls ---------------------------------------------------------------------------------------------------------------


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def stream():
    return torch.cuda.current_stream().cuda_stream


class Filled:
    """A cache with its definition beside it: sequences in pages of a scattered order."""

    def __init__(self, lens, nkvh, d, dtype, store, page=16, extra=0, seed=0):
        self.rng, self.dtype, self.store, self.page, self.nkvh, self.d = np.random.default_rng(seed), dtype, store, page, nkvh, d
        self.room = [-(-(n + extra) // page) for n in lens]
        pages = sum(self.room) + 3
        self.cache = llaisys.PagedKVCache.quantized(pages, nkvh, d, store=STORES[store], dtype=NAMES[dtype], page_size=page, max_seqs=len(lens) + 2,
                                                    max_pages_per_seq=max(self.room + [1]))
        order = self.rng.permutation(pages).tolist()
        self.seqs = []
        for n in self.room:
            self.seqs.append(self.cache.add_seq())
            self.cache.assign_pages(self.seqs[-1], [order.pop() for _ in range(n)])
        self.k = [Definition(nkvh, d, store) for _ in lens]
        self.v = [Definition(nkvh, d, store) for _ in lens]
        self.append([(i, 0, n) for i, n in enumerate(lens) if n])

    def rows(self, n):
        x = self.rng.standard_normal((n, self.nkvh, self.d)) * np.exp(self.rng.uniform(-2, 2, (n, 1, 1)))
        return torch.from_numpy(x).to(TORCH[self.dtype])

    def append(self, parts, k=None, v=None):
        """parts: (sequence, first position, count), one call."""
        if not parts:
            return
        n = sum(c for _, _, c in parts)
        k = self.rows(n) if k is None else k
        v = self.rows(n) if v is None else v
        seq = [self.seqs[i] for i, _, c in parts for _ in range(c)]
        pos = [at + r for _, at, c in parts for r in range(c)]
        self.cache.flush()
        self.cache.append_dev(0, k.cuda(), v.cuda(), i32(seq), i32(pos), n, stream())
        at = 0
        for i, first, c in parts:
            self.k[i].append(first, k[at:at + c].float().numpy())
            self.v[i].append(first, v[at:at + c].float().numpy())
            at += c

    def check_rows(self):
        """Every row read back equals the definition's."""
        for i, seq in enumerate(self.seqs):
            n = len(self.k[i].codes)
            if n == 0:
                continue
            got = [torch.full((n, self.nkvh, self.d), 7.0, dtype=TORCH[self.dtype], device="cuda") for _ in range(2)]
            self.cache.gather_dev(0, *got, i32([seq] * n), i32(range(n)), n, stream())
            for g, want in zip(got, (self.k[i], self.v[i])):
                w = torch.from_numpy(want.worth()).to(TORCH[self.dtype])
                assert torch.equal(torch.isnan(g.cpu()), torch.isnan(w))
                assert torch.equal(torch.nan_to_num(g.cpu().float()), torch.nan_to_num(w.float()))

    def check_attention(self, parts, nh, window=0, keep=0, factor=None, stride=0, chunks=False, order=None):
        """parts: (sequence, queries): the last tokens of each. Compares the call with the definition."""
        group_rows = [n for _, n in parts]
        total = sum(group_rows)
        q = torch.randn(total + 2, nh, self.d, generator=torch.Generator().manual_seed(5)).to(TORCH[self.dtype])
        width = stride or nh * self.d
        out = torch.full((total + 2, width), 9.0, dtype=TORCH[self.dtype], device="cuda")
        starts = np.concatenate([[0], np.cumsum(group_rows)])
        lens = [len(self.k[i].codes) for i, _ in parts]
        qd, ids, kv = q.cuda(), i32([self.seqs[i] for i, _ in parts]), i32(lens)
        scale = self.d ** -0.5
        kw = dict(n_seqs=len(parts), total_q=total, max_q_len=max(group_rows), max_kv_len=max(lens), nh=nh, scale=scale, stream=stream())
        f = None if factor is None else factor.cuda()
        self.cache.attention_dev(0, out, qd, ids, i32(starts) if chunks else None, kv, window=window, keep_first=keep, row_scale=f, row_stride=stride,
                                 **kw)
        got = out.cpu()
        assert (got[total:] == 9).all() and (got[:, nh * self.d:] == 9).all()  # rows behind the last sequence, and between rows
        got = got[:total, :nh * self.d].view(total, nh, self.d).double()
        for (i, n), at in zip(parts, starts):
            k, v = (torch.from_numpy(x.worth()).double() for x in (self.k[i], self.v[i]))
            qs = q[at:at + n].double()
            want, top, big = attention_f64(qs, k, v, len(k) - n, scale, window, keep)
            tol = tolerance(want, top, big, self.dtype, len(k), self.d)
            if factor is not None:
                want, tol = want * factor[at:at + n].double()[..., None], tol * factor[at:at + n].double().abs()[..., None]
            nan = torch.isnan(want)
            assert torch.equal(nan, torch.isnan(got[at:at + n]))
            worst = ((got[at:at + n] - want).abs() / tol)[~nan]
            assert worst.numel() == 0 or worst.max() <= 1, (i, float(worst.max()))


# ---- append --------------------------------------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("store", ["i8", "f8"])
@pytest.mark.parametrize("dtype,nkvh,d,page", [("bf16", 2, 128, 16), ("f16", 3, 64, 32), ("f32", 1, 96, 16), ("bf16", 5, 256, 64), ("f32", 2, 32, 48)])
def test_append_whole_and_in_pieces(cuda_device, store, dtype, nkvh, d, page):
    f = Filled([1, 15, 16, 17, 0, 40, 130], nkvh, d, dtype, store, page, extra=60)
    f.check_rows()
    # pieces that begin inside blocks, one token at a time, and over several blocks; then tokens written again
    f.append([(0, 1, 1), (1, 15, 20), (3, 17, 1), (4, 0, 5), (5, 40, 8)])
    f.append([(0, 2, 1), (4, 5, 1), (5, 48, 1), (6, 130, 33)])
    f.append([(6, 100, 3), (5, 0, 2), (3, 9, 4)])
    f.check_rows()
    f.cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("store", ["i8", "f8"])
def test_append_token_by_token(cuda_device, store):
    f = Filled([0, 3], 2, 64, "bf16", store, 16, extra=40)
    for t in range(37):
        f.append([(1, 3 + t, 1), (0, t, 1)])
    f.check_rows()


@pytest.mark.gpu
@pytest.mark.parametrize("store", ["i8", "f8"])
def test_append_zeros_extremes_and_what_is_not_finite(cuda_device, store):
    f = Filled([0, 0, 0, 0], 2, 32, "f32", store, 16, extra=48)
    zero = torch.zeros(20, 2, 32)
    f.append([(0, 0, 20)], zero, zero)
    f.append([(0, 20, 2)], torch.full((2, 2, 32), 1e-38), torch.full((2, 2, 32), 3e38))
    rows = f.rows(20)
    rows[3, 0, 5], rows[18, 1, 7] = torch.nan, -torch.inf
    f.append([(1, 0, 20)], rows, f.rows(20))
    f.append([(1, 20, 4)])   # behind a block that is lost
    f.append([(1, 0, 16)])   # written again from its first slot: sound again
    f.append([(2, 0, 5)])
    f.append([(2, 5, 2)], torch.full((2, 2, 32), torch.nan), f.rows(2))
    f.check_rows()


@pytest.mark.gpu
def test_append_skips_rows_without_sequence_and_flags_bad_ones(cuda_device):
    f = Filled([20, 20], 2, 64, "bf16", "i8", 16, extra=12)
    k = f.rows(6)
    f.cache.append_dev(0, k.cuda(), k.cuda(), i32([-1, f.seqs[0], f.seqs[0], -1, -1, -1]), i32([-1, 20, 21, -1, 5, 0]), 6, stream())
    f.k[0].append(20, k[1:3].float().numpy())
    f.v[0].append(20, k[1:3].float().numpy())
    f.cache.check()
    f.check_rows()
    for seq, pos in ((99, 0), (-2, 0), (0, -1), (0, 1 << 20)):
        f.cache.append_dev(0, k.cuda(), k.cuda(), i32([seq]), i32([pos]), 1, stream())
        with pytest.raises(llaisys.LlaisysError) as e:
            f.cache.check()
        assert e.value.status == Status.KERNEL
        out = torch.full((1, 2, 64), 7.0, dtype=torch.bfloat16, device="cuda")
        f.cache.gather_dev(0, out, out, i32([seq]), i32([pos]), 1, stream())
        assert (out == 7).all()
        with pytest.raises(llaisys.LlaisysError):
            f.cache.check()
    f.check_rows()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,store,nkvh,d", [("bf16", "i8", 4, 128), ("f16", "f8", 8, 64), ("f32", "i8", 4, 96), ("bf16", "f8", 3, 256)])
def test_append_of_many_rows_among_them_some_without_a_place(cuda_device, dtype, store, nkvh, d):
    """Runs that are skipped or flagged between runs that are stored, several to a warp: the others are what they are without them."""
    rng = np.random.default_rng(nkvh)
    lens = rng.integers(0, 60, 90)
    f = Filled(lens.tolist(), nkvh, d, dtype, store, extra=40)
    seq, pos, good = [], [], []
    for i, held in enumerate(lens.tolist()):
        n = int(rng.integers(1, 40))
        good.append((i, held, n, len(seq)))
        seq += [f.seqs[i]] * n
        pos += range(held, held + n)
        for _ in range(int(rng.integers(1, 3))):
            m = int(rng.integers(1, 20))
            at, s = [(0, 99), (1 << 20, f.seqs[i]), (7, -1), (-1, -1), (3, 1 << 30)][int(rng.integers(0, 5))]
            seq += [s] * m
            pos += [at] * m if at < 0 else range(at, at + m)
    rows = len(seq)
    assert rows * 2 * nkvh > 64 * torch.cuda.get_device_properties(0).multi_processor_count  # the form of many rows
    k, v = f.rows(rows), f.rows(rows)
    bad = torch.ones(rows, dtype=torch.bool)
    for _, _, n, at in good:
        bad[at:at + n] = False
    k[bad] *= 1000  # what would be seen anywhere else
    v[bad] *= 1000
    f.cache.append_dev(0, k.cuda(), v.cuda(), i32(seq), i32(pos), rows, stream())
    for i, held, n, at in good:
        f.k[i].append(held, k[at:at + n].float().numpy())
        f.v[i].append(held, v[at:at + n].float().numpy())
    with pytest.raises(llaisys.LlaisysError) as e:
        f.cache.check()
    assert e.value.status == Status.KERNEL
    f.check_rows()


@pytest.mark.gpu
@pytest.mark.parametrize("store", ["i8", "f8"])
@pytest.mark.parametrize("dtype,nkvh,d,page", [("bf16", 2, 128, 16), ("f16", 8, 32, 48), ("f32", 4, 64, 32), ("f32", 1, 256, 16)])
def test_many_rows_in_a_call(cuda_device, dtype, store, nkvh, d, page):
    """Several thousand rows at a time, appended from inside blocks on and read back in one call: in order, out of order, and with rows in between that
    do not exist. Every number equals the definition's."""
    rng = np.random.default_rng(d)
    few = 64 * torch.cuda.get_device_properties(0).multi_processor_count // (2 * nkvh)  # rows up to which a warp takes one
    lens = [int(x) for x in rng.integers(0, 40, 150)] + [few, 300]
    f = Filled(lens, nkvh, d, dtype, store, page, extra=2 * few)
    new = [int(x) for x in rng.integers(0, 50, 150)] + [few + 13, 7]
    f.append([(i, n, m) for i, (n, m) in enumerate(zip(lens, new)) if m])
    f.append([(i, n + m, 1) for i, (n, m) in enumerate(zip(lens, new))])
    seq = np.concatenate([[s] * (n + m + 1) for s, n, m in zip(f.seqs, lens, new)])
    pos = np.concatenate([np.arange(n + m + 1) for n, m in zip(lens, new)])
    assert len(seq) > few
    wants = [torch.from_numpy(np.concatenate([x.worth() for x in side])).to(TORCH[dtype]) for side in (f.k, f.v)]
    mixed = rng.permutation(len(seq))
    gaps = np.sort(rng.choice(len(seq), 200, replace=False))
    for order, bad in ((np.arange(len(seq)), False), (mixed, False), (np.arange(len(seq)), True)):
        s, p = seq[order].copy(), pos[order].copy()
        if bad:
            s[gaps[:100]], p[gaps[100:]] = 99999, np.where(gaps[100:] % 2, -1, 1 << 22)
        got = [torch.full((len(seq), nkvh, d), 7.0, dtype=TORCH[dtype], device="cuda") for _ in range(2)]
        f.cache.gather_dev(0, *got, i32(s), i32(p), len(seq), stream())
        for g, want in zip(got, wants):
            want = want[torch.from_numpy(order)]
            if bad:
                want[torch.from_numpy(gaps)] = 7.0
            assert torch.equal(g.cpu(), want)
        if bad:
            with pytest.raises(llaisys.LlaisysError):
                f.cache.check()
    f.cache.check()


@pytest.mark.gpu
def test_host_forms_fork_and_prefix(cuda_device):
    f = Filled([37, 5], 2, 64, "f16", "i8", 16, extra=20)
    k, v = f.rows(4), f.rows(4)
    kd, vd = k.cuda(), v.cuda()
    f.cache.append(0, kd, vd, [f.seqs[0]] * 3 + [f.seqs[1]], [37, 38, 39, 5])
    for i, part in ((0, slice(0, 3)), (1, slice(3, 4))):
        f.k[i].append((37, 5)[i], k[part].float().numpy())
        f.v[i].append((37, 5)[i], v[part].float().numpy())
    out = [torch.empty(40, 2, 64, dtype=torch.float16, device="cuda") for _ in range(2)]
    f.cache.gather(0, f.seqs[0], 40, *out)
    torch.cuda.synchronize()
    assert torch.equal(out[0].cpu().float(), torch.from_numpy(f.k[0].worth()).half().float())
    child = f.cache.fork(f.seqs[0], 39)  # the last page is copied, scales and all
    again = [torch.empty(39, 2, 64, dtype=torch.float16, device="cuda") for _ in range(2)]
    f.cache.gather(0, child, 39, *again)
    torch.cuda.synchronize()
    assert torch.equal(again[0], out[0][:39]) and torch.equal(again[1], out[1][:39])
    for seqs, pos in (([0, 0], [41, 40]), ([0, 1, 0], [41, 6, 42]), ([0, 0], [41, 41])):
        with pytest.raises(llaisys.LlaisysError) as e:
            f.cache.append(0, kd, vd, seqs, pos)
        assert e.value.status == Status.INVALID
    # decode, chunk and partial results through the host forms
    q = torch.randn(2, 4, 64, dtype=torch.float16, device="cuda")
    o, part = torch.empty_like(q), torch.empty(2, 4, 66, device="cuda")
    f.cache.decode(0, o, q, f.seqs, [40, 6], 4, 0.125)
    f.cache.decode_partial(0, part, q, f.seqs, [40, 6], 4, 0.125)
    torch.cuda.synchronize()
    assert torch.allclose(part[..., :64], o.float(), rtol=2.0 ** -10, atol=1e-6)
    for i, n in enumerate((40, 6)):
        ks = torch.from_numpy(f.k[i].worth()).double().repeat_interleave(2, 1)
        s = torch.einsum("hd,jhd->hj", q[i].cpu().double(), ks) * 0.125
        assert torch.allclose(part[i, :, 64].cpu().double(), s.amax(-1), rtol=1e-4, atol=1e-4)
        assert torch.allclose(part[i, :, 65].cpu().double(), (s - s.amax(-1, keepdim=True)).exp().sum(-1), rtol=1e-3)


# ---- attention -----------------------------------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("store", ["i8", "f8"])
@pytest.mark.parametrize("dtype,nh,nkvh,d,page", [("bf16", 12, 2, 128, 16), ("f16", 8, 8, 64, 32), ("f32", 6, 3, 96, 16), ("bf16", 40, 2, 256, 64),
                                                  ("f32", 4, 1, 128, 16), ("f16", 32, 1, 32, 48)])
def test_decode(cuda_device, store, dtype, nh, nkvh, d, page):
    f = Filled([1, 2, 15, 16, 17, 100, 333, 2050], nkvh, d, dtype, store, page)
    f.check_attention([(i, 1) for i in (3, 0, 7, 1, 2, 6, 4, 5)], nh)
    f.cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("store", ["i8", "f8"])
@pytest.mark.parametrize("dtype,nh,nkvh,d,page", [("bf16", 12, 2, 128, 16), ("f16", 8, 2, 64, 32), ("f32", 6, 3, 96, 16), ("bf16", 17, 1, 128, 16),
                                                  ("f32", 4, 4, 256, 64), ("f16", 32, 8, 128, 16)])
def test_chunks(cuda_device, store, dtype, nh, nkvh, d, page):
    f = Filled([1, 5, 16, 70, 200, 513, 1029], nkvh, d, dtype, store, page)
    f.check_attention([(6, 300), (0, 1), (5, 17), (1, 5), (2, 2), (3, 33), (4, 200)], nh, chunks=True)
    f.check_attention([(6, 1), (4, 1)], nh, chunks=True)
    f.cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("window,keep", [(1, 0), (7, 3), (16, 16), (100, 20), (5000, 4), (33, 100)])
@pytest.mark.parametrize("dtype,store,d", [("bf16", "i8", 128), ("f32", "f8", 64), ("f16", "f8", 128)])
def test_windows_factors_and_strides(cuda_device, window, keep, dtype, store, d):
    f = Filled([1, 40, 130, 777], 2, d, dtype, store)
    factor = torch.randn(400, 8, generator=torch.Generator().manual_seed(3))
    f.check_attention([(3, 1), (1, 1), (0, 1), (2, 1)], 8, window=window, keep=keep, factor=factor[:4], stride=8 * d + 8)
    f.check_attention([(3, 260), (0, 1), (2, 100), (1, 39)], 8, window=window, keep=keep, factor=factor, stride=8 * d + 8, chunks=True)


@pytest.mark.gpu
@pytest.mark.parametrize("store", ["i8", "f8"])
@pytest.mark.parametrize("dtype,nh,nkvh,d,page", [("bf16", 12, 2, 128, 16), ("f16", 32, 8, 64, 32), ("bf16", 16, 1, 128, 64), ("f16", 8, 8, 128, 16),
                                                  ("bf16", 24, 1, 64, 16)])
def test_long_chunks(cuda_device, store, dtype, nh, nkvh, d, page):
    f = Filled([4, 900, 300, 513, 1029, 2050], nkvh, d, dtype, store, page)
    parts = [(3, 513), (0, 3), (5, 700), (1, 900), (4, 1), (2, 299)]
    f.check_attention(parts, nh, chunks=True)
    assert f.cache.last_kernel() == llaisys.Kernel.EIGHT_BIT_TC
    factor = torch.randn(2416, nh, generator=torch.Generator().manual_seed(3))
    for window, keep in ((1, 0), (100, 17), (600, 300)):
        f.check_attention(parts, nh, window=window, keep=keep, factor=factor, stride=nh * d + 16, chunks=True)
        assert f.cache.last_kernel() == llaisys.Kernel.EIGHT_BIT_TC
    f.cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("window", [0, 40])
def test_long_chunks_longer_than_their_sequences_and_lost_blocks(cuda_device, window):
    nh, d = 8, 128
    f = Filled([700, 260, 1], 2, d, "bf16", "i8", extra=16)
    bad = f.rows(1)
    bad[0, 0, 3] = torch.inf
    f.append([(0, 400, 1)], bad, f.rows(1))
    f.append([(1, 17, 1)], f.rows(1), bad)
    q = torch.randn(2700, nh, d, generator=torch.Generator().manual_seed(5)).bfloat16()
    starts, lens = [0, 900, 1800, 2600, 2600], [700, 260, 1, 0]
    out = torch.full((2700, nh, d), 9.0, dtype=torch.bfloat16, device="cuda")
    qd = q.cuda()
    ids = i32([*f.seqs, 0])
    f.cache.attention_dev(0, out, qd, ids, i32(starts), i32(lens), n_seqs=4, total_q=2600, max_q_len=900, max_kv_len=700, nh=nh, scale=-0.05,
                          stream=stream(), window=window)
    assert f.cache.last_kernel() == llaisys.Kernel.EIGHT_BIT_TC
    got = out.cpu().double()
    assert (got[2600:] == 9).all()
    for i in range(3):
        n, at = starts[i + 1] - starts[i], starts[i]
        k, v = (torch.from_numpy(x.worth()).double() for x in (f.k[i], f.v[i]))
        lead = n - lens[i]  # queries in front of the first token
        assert (got[at:at + lead] == 0).all()
        want, top, big = attention_f64(q[at + lead:at + n].double(), k, torch.nan_to_num(v), 0, -0.05, window)
        # values of a lost block reach whoever sees one of its keys
        t, j = torch.arange(lens[i])[:, None], torch.arange(lens[i])[None, :]
        seen = (j <= t) & ((t - j < window) if window else True)
        lost = torch.isnan(v).any(-1)  # [token, kv head]
        hit = (seen.double() @ lost.double()).repeat_interleave(nh // 2, 1) > 0
        want = torch.where(hit[..., None], torch.nan, want)
        part = got[at + lead:at + n]
        nan = torch.isnan(want)
        assert torch.equal(nan, torch.isnan(part))
        tol = tolerance(torch.nan_to_num(want), torch.nan_to_num(top), torch.nan_to_num(big), "bf16", lens[i], d)
        assert ((part - want).abs() <= tol)[~nan].all()
    f.cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_that_see_nothing_and_lost_blocks(cuda_device, dtype):
    f = Filled([40, 300], 2, 128, dtype, "i8")
    q = torch.randn(3, 4, 128, device="cuda").to(TORCH[dtype])
    out = torch.full_like(q, 9.0)
    f.cache.decode_dev(0, out, q, i32([f.seqs[0], f.seqs[1], f.seqs[0]]), i32([40, 0, 0]), 3, 300, 4, 0.1, stream())
    assert (out[1:] == 0).all() and not (out[0] == 0).all()
    # more queries than tokens: the first ones see nothing
    out.fill_(9.0)
    f.cache.prefill_dev(0, out, q, i32([f.seqs[0]]), i32([0, 3]), i32([2]), 1, 3, 3, 2, 4, 0.1, stream())
    assert (out[0] == 0).all() and not (out[1] == 0).all()
    # a NaN in a block: queries that read the block are NaN, the others are not
    bad = f.rows(1)
    bad[0, 1, 5] = torch.nan
    f.append([(1, 200, 1)], bad, f.rows(1))
    f.check_attention([(1, 1)], 4)
    f.check_attention([(1, 1)], 4, window=80)
    f.check_attention([(1, 1)], 4, window=80, keep=16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,nh,nkvh,d,store", [("bf16", 12, 2, 128, "i8"), ("f16", 32, 8, 64, "f8"), ("f32", 8, 2, 96, "i8"), ("bf16", 20, 1, 256, "f8")])
@pytest.mark.parametrize("window", [0, 50])
def test_sequences_that_do_not_exist_beside_others(cuda_device, dtype, nh, nkvh, d, store, window):
    """Queries of no sequence between others: flagged, and the others' answers are what they are without them."""
    lens = [1, 70, 333, 16, 900, 45, 2050, 300]
    f = Filled(lens, nkvh, d, dtype, store)
    ids = [x for s in f.seqs for x in (s, 99)]
    for count in (1, 5):  # single queries; chunks
        kv = [x for n in lens for x in (max(n, count), 700)]
        q = torch.randn(len(ids) * count, nh, d, generator=torch.Generator().manual_seed(5)).to(TORCH[dtype])
        qd, out = q.cuda(), torch.full((len(ids) * count, nh, d), 9.0, dtype=TORCH[dtype], device="cuda")
        starts = i32(range(0, len(ids) * count + 1, count)) if count > 1 else None
        f.cache.attention_dev(0, out, qd, i32(ids), starts, i32(kv), n_seqs=len(ids), total_q=len(ids) * count, max_q_len=count, max_kv_len=2050, nh=nh,
                              scale=d ** -0.5, stream=stream(), window=window)
        assert f.cache.last_kernel() == llaisys.Kernel.EIGHT_BIT
        got = out.cpu().view(len(ids), count, nh, d).double()
        assert (got[1::2] == 0).all()
        for i, n in enumerate(lens):
            if n < count:
                continue
            k, v = (torch.from_numpy(x.worth()).double() for x in (f.k[i], f.v[i]))
            want, top, big = attention_f64(q[2 * i * count:(2 * i + 1) * count].double(), k, v, n - count, d ** -0.5, window)
            assert ((got[2 * i] - want).abs() <= tolerance(want, top, big, dtype, n, d)).all(), (count, i)
        with pytest.raises(llaisys.LlaisysError) as e:
            f.cache.check()
        assert e.value.status == Status.KERNEL


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,nh,nkvh,d,page,store", [("bf16", 12, 2, 128, 16, "i8"), ("f16", 32, 8, 64, 32, "f8"), ("f32", 6, 3, 96, 16, "i8"),
                                                        ("bf16", 16, 1, 128, 64, "f8"), ("f16", 4, 4, 256, 16, "i8")])
@pytest.mark.parametrize("window", [0, 150])
def test_pages_that_do_not_exist(cuda_device, dtype, nh, nkvh, d, page, store, window):
    """Their tokens are nobody's keys, whichever kernel serves the call; so are all tokens of a sequence that does not exist. Both are flagged."""
    lens = [700, 64, 333, 1029]
    f = Filled(lens, nkvh, d, dtype, store, page)
    stride = max(f.room)
    lost = [[0, 3, 4, 10], [], [f.room[2] - 1], list(range(f.room[3] // 2, f.room[3] - 1))]
    table = np.zeros((len(lens) + 2, stride), np.int32)
    for s, pages, gone in zip(f.seqs, f.room, lost):
        table[s, :pages] = f.cache.seq_pages(s)
        table[s, [e for e in gone if e < pages]] = -1 if s % 2 else 1 << 20
    torch.cuda.synchronize()
    llaisys.RuntimeAPI(llaisys.DeviceType.NVIDIA).memcpy_sync(f.cache.block_table_ptr(), table.ctypes.data, table.nbytes, llaisys.MemcpyKind.H2D)
    ids = [*f.seqs, 77]
    for counts, tc in (([1] * 5, False), ([3, 1, 5, 2, 4], False), ([300, 64, 200, 513, 90], d in (64, 128) and dtype != "f32")):
        starts, total = np.concatenate([[0], np.cumsum(counts)]), sum(counts)
        q = torch.randn(total, nh, d, generator=torch.Generator().manual_seed(5)).to(TORCH[dtype])
        qd, out = q.cuda(), torch.full((total, nh, d), 9.0, dtype=TORCH[dtype], device="cuda")
        f.cache.attention_dev(0, out, qd, i32(ids), i32(starts) if total > 5 else None, i32([*lens, 500]), n_seqs=5, total_q=total, max_q_len=max(counts),
                              max_kv_len=max(lens), nh=nh, scale=d ** -0.5, stream=stream(), window=window)
        assert (f.cache.last_kernel() == llaisys.Kernel.EIGHT_BIT_TC) == tc
        got = out.cpu().double()
        assert (got[starts[4]:] == 0).all()
        for i, n in enumerate(lens):
            rows = slice(starts[i], starts[i + 1])
            k, v = (torch.from_numpy(x.worth()).double().repeat_interleave(nh // nkvh, 1) for x in (f.k[i], f.v[i]))
            t, j = torch.arange(n - counts[i], n)[:, None], torch.arange(n)[None]
            seen = (j <= t) & (t - j < (window or n)) & ~torch.isin(j // page, torch.tensor(lost[i], dtype=torch.int64))
            x = torch.einsum("thd,jhd->htj", q[rows].double(), k) * d ** -0.5
            p = torch.where(seen.any(-1)[None, :, None], torch.softmax(x.masked_fill(~seen, -torch.inf), -1), 0.0)
            big = (torch.einsum("thd,jhd->htj", q[rows].double().abs(), k.abs()) * d ** -0.5).masked_fill(~seen, 0).amax(-1).T
            top = torch.where(seen[None], v.abs().amax(-1).T[:, None, :], 0).amax(-1).T
            want = torch.einsum("htj,jhd->thd", p, v)
            assert ((got[rows] - want).abs() <= tolerance(want, top, big, dtype, n, d)).all(), (counts, i)
        with pytest.raises(llaisys.LlaisysError) as e:
            f.cache.check()
        assert e.value.status == Status.KERNEL
    # a sequence that does not exist and holds nothing: nothing is looked up
    for starts in (None, i32([0, 1]), i32([0, 1000])):
        out = torch.full((1000, nh, d), 9.0, dtype=TORCH[dtype], device="cuda")
        n = 1 if starts is None else int(starts[1])
        f.cache.attention_dev(0, out, torch.ones_like(out), i32([77]), starts, i32([0]), n_seqs=1, total_q=n, max_q_len=n, max_kv_len=max(lens), nh=nh,
                              scale=1.0, stream=stream(), window=window)
        assert (out[:n] == 0).all() and (out[n:] == 9).all()
        f.cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,nh,nkvh,d", [("bf16", 2, 2, 128), ("f16", 4, 1, 64), ("f32", 12, 2, 96), ("bf16", 16, 1, 256)])
def test_tables_that_are_full(cuda_device, dtype, nh, nkvh, d):
    """Sequences that end in the last block of their tables: nothing behind it is looked up."""
    f = Filled([160, 159, 158, 157, 156, 145, 144], nkvh, d, dtype, "i8")
    parts = [(i, 1) for i in range(7)]
    f.check_attention(parts, nh)
    f.check_attention(parts, nh, window=40, keep=20)
    for n in (1, 2, 3, 5, 140):
        f.check_attention([(i, n) for i, _ in parts], nh, chunks=True)
        f.check_attention([(i, n) for i, _ in parts], nh, window=20, keep=3, chunks=True)
    f.cache.check()


@pytest.mark.gpu
def test_one_long_sequence(cuda_device):
    f = Filled([70001], 1, 64, "bf16", "i8")
    f.check_attention([(0, 1)], 8)
    f.check_attention([(0, 9)], 8, chunks=True)


@pytest.mark.gpu
def test_values_of_very_different_size(cuda_device):
    """Blocks whose scales are far apart, and queries far from one."""
    f = Filled([0], 2, 64, "f32", "i8", extra=200)
    k, v = f.rows(180), f.rows(180)
    v *= torch.exp2(torch.linspace(-60, 40, 180))[:, None, None]
    k *= torch.exp2(torch.linspace(-90, -3, 180))[:, None, None]
    f.append([(0, 0, 180)], k, v)
    f.check_rows()
    f.check_attention([(0, 1)], 4)
    f.check_attention([(0, 60)], 4, chunks=True)


def constant_rows(seqs, tokens, nkvh, d, dtype, store, k_of, v_of):
    """A cache of sequences whose token t has the numbers k_of(t) and v_of(t) in every dim."""
    pages = -(-tokens // 16)
    cache = llaisys.PagedKVCache.quantized(seqs * pages, nkvh, d, store=STORES[store], dtype=NAMES[dtype], max_seqs=seqs, max_pages_per_seq=pages)
    t = torch.arange(tokens, device="cuda")
    k, v = (of(t).to(TORCH[dtype])[:, None, None].expand(-1, nkvh, d).contiguous() for of in (k_of, v_of))
    for _ in range(seqs):
        s = cache.add_seq()
        cache.reserve(s, tokens)
        cache.flush()
        cache.append_dev(0, k, v, torch.full((tokens,), s, dtype=torch.int32, device="cuda"), t.int(), tokens, stream())
    return cache


@pytest.mark.gpu
@pytest.mark.parametrize("store", ["i8", "f8"])
@pytest.mark.parametrize("dtype,nh", [("bf16", 4), ("f32", 4), ("f16", 16)])
def test_values_that_are_zero_for_long(cuda_device, dtype, store, nh):
    """20000 tokens of value 0 and equal scores, then 1000 of value 4: the row's sum counts them all."""
    n, last, d = 21000, 1000, 64
    cache = constant_rows(1, n, 1, d, dtype, store, lambda t: 0.0 * t, lambda t: 4.0 * (t >= n - last))
    q = torch.ones(1, nh, d, dtype=TORCH[dtype], device="cuda")
    out, part = torch.empty_like(q), torch.empty(1, nh, d + 2, device="cuda")
    # weights are off by 2^-11 (their sum and theirs with the values), the values' code by nothing but the scale's rounding
    tol = dict(rtol=torch.finfo(TORCH[dtype]).eps / 2 + 2.0 ** -9, atol=0)
    for held in (n, n - last):
        value = 4 * last / n if held == n else 0
        cache.decode_dev(0, out, q, i32([0]), i32([held]), 1, held, nh, 0.1, stream())
        cache.decode_partial_dev(0, part, q, i32([0]), i32([held]), 1, held, nh, 0.1, stream())
        assert torch.allclose(out.float().cpu(), torch.tensor(float(value)), **tol)
        assert torch.allclose(part[..., :d].cpu(), torch.tensor(float(value)), **tol)
        assert (part[..., d] == 0).all() and torch.allclose(part[..., d + 1].cpu(), torch.tensor(float(held)), rtol=1e-5)
    cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("store", ["i8", "f8"])
def test_long_chunks_behind_values_that_are_zero_for_long(cuda_device, store):
    """The same for chunks, a whole tile a CTA, with scores that rise as far as the maximum may lag behind them."""
    n, rows, d, seqs = 16384, 64, 64, 4
    nkvh = torch.cuda.get_device_properties(0).multi_processor_count // seqs
    cache = constant_rows(seqs, n, nkvh, d, "bf16", store, lambda t: 1.0 * (t >= 128), lambda t: 4.0 * (t >= n - 128))
    q = torch.ones(seqs * rows, 4 * nkvh, d, dtype=torch.bfloat16, device="cuda")
    out = torch.empty_like(q)
    rise = 7.9  # a key of ones, in log2 units
    cache.prefill_dev(0, out, q, i32(range(seqs)), i32(range(0, seqs * rows + 1, rows)), i32([n] * seqs), seqs, seqs * rows, rows, n, 4 * nkvh,
                      rise * np.log(2) / d, stream())
    assert cache.last_kernel() == llaisys.Kernel.EIGHT_BIT_TC
    seen = n - rows + 1 + torch.arange(rows).double()
    want = 4 * (seen - (n - 128)) * 2 ** rise / ((seen - 128) * 2 ** rise + 128)
    got = out.view(seqs, rows, -1).cpu().double()
    assert ((got - want[None, :, None]).abs() <= want[None, :, None] * (2.0 ** -8 + 2.0 ** -9)).all()
    cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("store", ["i8", "f8"])
@pytest.mark.parametrize("dtype,nh", [("bf16", 4), ("f32", 4), ("bf16", 16)])
def test_queries_at_the_end_of_their_range(cuda_device, dtype, store, nh):
    """Keys that are zero have score 0 whatever the queries: the mean of the values."""
    n, d = 400, 64
    cache = constant_rows(1, n, 1, d, dtype, store, lambda t: 0.0 * t, lambda t: 1.0 + t // 16 % 2)
    q = torch.full((n, nh, d), torch.finfo(TORCH[dtype]).max, dtype=TORCH[dtype], device="cuda")
    q[::3] = -2.0 ** 121
    out = torch.empty_like(q)
    tol = torch.finfo(TORCH[dtype]).eps / 2 + (2.0 ** -20 if dtype == "f32" else 2.0 ** -11 * 1.01)
    for rows in (1, 3, n):
        starts = None if rows == 1 else i32([0, rows])
        cache.attention_dev(0, out, q, i32([0]), starts, i32([n]), n_seqs=1, total_q=rows, max_q_len=rows, max_kv_len=n, nh=nh, scale=1.0,
                            stream=stream())
        value = (1.0 + torch.arange(n).double() // 16 % 2).cumsum(0) / torch.arange(1, n + 1)
        assert ((out[:rows].cpu().double() - value[n - rows:, None, None]).abs() <= 2 * tol).all(), rows
    cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,nh,d", [("f16", 4, 64), ("bf16", 4, 128), ("f16", 16, 64), ("bf16", 2, 256)])
def test_long_sums_of_integers_do_not_drift(cuda_device, dtype, nh, d):
    """Means of 60000 values, 15000 of them to a warp, all of one scale s and of weight w = f16(s). Besides w, which is off by 2^-11 of itself, only sums
    are rounded, by 2^-23 of the sum an addition of 16 tokens: in 256 tokens, 16 additions to at most 255 w a token and 16 to w a token that count 128
    times; and n / 16 additions to what was there, which after t codes of either sign (59 rms) is not over 4 * 59 sqrt(t) w: 236 / 16 * 2 / 3 sqrt(n) of
    them a token. A few more where parts join, of the mean itself, which is below one code."""
    n, seqs = 60000, 3 * torch.cuda.get_device_properties(0).multi_processor_count
    pages = n // 16
    cache = llaisys.PagedKVCache.quantized(pages, 1, d, dtype=NAMES[dtype], max_seqs=1, max_pages_per_seq=pages)
    v = (torch.randint(-100, 101, (n, 1, d), generator=torch.Generator().manual_seed(3)) * 1.4719).to(TORCH[dtype])
    v[::32, 0, 0], v[16::32, 0, 0] = 187, -187  # the largest of every block
    values = Definition(1, d, "i8")
    values.append(0, v.float().numpy())
    unit = 187 / 127
    cache.reserve(cache.add_seq(), n)
    cache.flush()
    cache.append_dev(0, torch.zeros(n, 1, d, dtype=TORCH[dtype], device="cuda"), v.cuda(), i32([0] * n), i32(range(n)), n, stream())
    q = torch.randn(seqs, nh, d, generator=torch.Generator().manual_seed(4)).to(TORCH[dtype]).cuda()
    part = torch.empty(seqs, nh, d + 2, device="cuda")
    cache.decode_partial_dev(0, part, q, i32([0] * seqs), i32([n] * seqs), seqs, n, nh, 0.1, stream())
    want = torch.from_numpy(values.worth()).double()[:, 0].mean(0)
    off = (part[..., :d].cpu().double() - want).abs() - want.abs() * 2.0 ** -11
    assert want.abs().max() < unit
    assert off.max() <= (16 * (255 + 128) + 236 / 24 * 15000 ** 0.5 + 64) * 2.0 ** -23 * unit, off.max() / unit * 2.0 ** 23
    cache.check()


# ---- a step, planned and run ----------------------------------------------------------------------------------------------


def plan_reference(ids, held, new, page, rows, free, table):
    table, q, p, at = table.copy(), [0], [0], 0
    seqs, pos, slots = [], [], []
    for i, h, n in zip(ids, held, new):
        for e in range(-(-h // page), -(-(h + n) // page)):
            table[i, e] = free[at]
            at += 1
        for t in range(h, h + n):
            seqs.append(i)
            pos.append(t)
            slots.append(int(table[i, t // page]) * page + t % page)
        q.append(q[-1] + n)
        p.append(p[-1] + -(-(h + n) // page))
    pad = [-1] * (rows - len(seqs))
    return dict(q_starts=q, kv_lens=[h + n for h, n in zip(held, new)], page_starts=p, row_seqs=seqs + pad, row_positions=pos + pad,
                row_slots=slots + pad, status=[at, 0]), table


def run_plan(ids, held, new, page, rows, free, table, null_ids=False, skip=()):
    n = len(held)
    out = dict(q_starts=torch.full((n + 1,), -7, dtype=torch.int32, device="cuda"), kv_lens=torch.full((n,), -7, dtype=torch.int32, device="cuda"),
               page_starts=torch.full((n + 1,), -7, dtype=torch.int32, device="cuda"), row_seqs=torch.full((rows,), -7, dtype=torch.int32, device="cuda"),
               row_positions=torch.full((rows,), -7, dtype=torch.int32, device="cuda"),
               row_slots=torch.full((rows,), -7, dtype=torch.int64, device="cuda"), status=torch.full((2,), -7, dtype=torch.int32, device="cuda"))
    t = torch.from_numpy(table).cuda() if table is not None else None
    f = i32(free) if free is not None else None
    hd, nd, idd = i32(held), i32(new), None if null_ids else i32(ids)
    llaisys.paged_plan_dev(stream=stream(), seq_ids_dev=idd, held_dev=hd, new_dev=nd, n_seqs=n, page_size=page, n_rows=rows, free_pages_dev=f,
                           n_free=0 if free is None else len(free), block_table_dev=t, table_rows=0 if t is None else t.shape[0],
                           table_stride=0 if t is None else t.shape[1], **{f"{k}_dev": None if k in skip else v for k, v in out.items()})
    return {k: v.cpu().numpy() for k, v in out.items()}, None if t is None else t.cpu().numpy()


@pytest.mark.gpu
@pytest.mark.parametrize("n,low,high,short,long,page", [(1, 0, 0, 1, 1, 16), (1, 5, 5, 0, 0, 16), (7, 0, 40, 0, 3, 16), (64, 1, 4096, 1, 1, 16),
                                                        (333, 0, 900, 0, 200, 32), (1024, 0, 50, 1, 2, 1), (2500, 0, 300, 0, 60, 48),
                                                        (3, 0, 100, 20000, 30000, 16), (40000, 0, 20, 0, 2, 16)])
def test_plan(cuda_device, n, low, high, short, long, page):
    rng = np.random.default_rng(n)
    held, new = rng.integers(low, high + 1, n), rng.integers(short, long + 1, n)
    stride = max(1, int((-(-(held + new) // page)).max()))
    ids = rng.permutation(n + 3)[:n]
    table = rng.integers(0, 9999, (n + 3, stride)).astype(np.int32)
    grown = int((-(-(held + new) // page) + -held // page).sum())
    free = rng.permutation(grown + 5).astype(np.int32)
    rows = int(new.sum()) + 70
    got, t = run_plan(ids, held, new, page, rows, free, table)
    want, w = plan_reference(ids.tolist(), held.tolist(), new.tolist(), page, rows, free, table)
    for key, value in want.items():
        assert np.array_equal(got[key], value), key
    assert np.array_equal(t, w)


@pytest.mark.gpu
def test_plan_what_cannot_be_done(cuda_device):
    table = np.arange(40, dtype=np.int32).reshape(4, 10)
    # too few pages: none is taken, rows on pages that are there have slots
    got, t = run_plan([0, 1], [10, 16], [10, 20], 16, 40, [90, 91], table)
    assert np.array_equal(t, table) and got["status"].tolist() == [0, 1]
    assert got["row_slots"][:10].tolist() == [0 * 16 + 10 + i for i in range(6)] + [-1] * 4 and (got["row_slots"][10:] == -1).all()
    assert got["q_starts"].tolist() == [0, 10, 30] and got["kv_lens"].tolist() == [20, 36]
    # rows that do not fit
    got, t = run_plan([0, 1, 2], [0, 0, 0], [5, 6, 7], 16, 8, None, table)
    assert got["q_starts"].tolist() == [0, 5, 8, 8] and got["status"].tolist() == [0, 2] and got["row_positions"].tolist() == [0, 1, 2, 3, 4, 0, 1, 2]
    # counts that are none, rows outside the table, requests longer than their row
    got, t = run_plan([0, 1, 7, 3], [-1, 2 ** 31 - 2, 3, 150], [4, 5, 2, 20], 16, 30, [50, 51, 52], table)
    assert got["status"].tolist() == [0, 4 | 8] and got["q_starts"].tolist() == [0, 0, 0, 2, 22]
    assert got["row_slots"][:2].tolist() == [-1, -1] and got["row_slots"][2:12].tolist() == [39 * 16 + 6 + i for i in range(10)]
    assert (got["row_slots"][12:] == -1).all() and np.array_equal(t, table)
    # nobody
    got, t = run_plan([], [], [], 16, 3, [1], table)
    assert got["q_starts"].tolist() == [0] and got["row_seqs"].tolist() == [-1] * 3 and got["status"].tolist() == [0, 0]
    # no table, no ids, outputs left out
    got, _ = run_plan(None, [4, 0], [1, 2], 16, 4, None, None, null_ids=True, skip=("row_slots", "page_starts", "status"))
    assert got["row_seqs"].tolist() == [0, 1, 1, -1] and got["row_positions"].tolist() == [4, 0, 1, -1] and (got["row_slots"] == -7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("free,new,flags", [([], [20, 14, 7, 30, 8], 1), ([11, 12, 13], [20, 14, 7, 30, 8], 1), ([11, 12, 13, 14], [20, 30, 7, 30, 8], 8),
                                            ([11, 12, 13], [20, 30, 7, 30, 8], 9)])
@pytest.mark.parametrize("slots", [False, True])
def test_plan_rows_without_a_page_are_not_appended(cuda_device, free, new, flags, slots):
    """Too few free pages, a request longer than its row of the table: the step's append leaves alone what the entries behind the requests' pages name."""
    lens = [20, 33, 16, 5, 40]
    f = Filled(lens, 2, 64, "bf16", "i8")
    stride, total = max(f.room), sum(new)
    table = np.zeros((len(lens) + 2, stride), np.int32)  # as the cache's: page 0 behind a sequence's last one
    for s, n in zip(f.seqs, f.room):
        table[s, :n] = f.cache.seq_pages(s)
    t, fr = torch.from_numpy(table).cuda(), i32(free + [0])
    seqs, pos = (torch.full((total + 5,), 7, dtype=torch.int32, device="cuda") for _ in range(2))
    status, at = i32([9, 9]), torch.full((total + 5,), 7, dtype=torch.int64, device="cuda")
    ids, hd, nd = i32(f.seqs), i32(lens), i32(new)
    llaisys.paged_plan_dev(stream=stream(), seq_ids_dev=ids, held_dev=hd, new_dev=nd, n_seqs=len(lens), page_size=16, n_rows=total + 5, free_pages_dev=fr,
                           n_free=len(free), block_table_dev=t, table_rows=len(table), table_stride=stride, row_seqs_dev=seqs, row_positions_dev=pos,
                           row_slots_dev=at if slots else None, status_dev=status)
    k, v = f.rows(total + 5), f.rows(total + 5)
    grown = flags == 8
    assert status.tolist() == [4 if grown else 0, flags]
    want_seqs, want_pos, row = [], [], 0
    for i, (s, held, n) in enumerate(zip(f.seqs, lens, new)):
        room = 16 * (stride if grown and held + n <= 16 * stride else f.room[i])
        kept = min(n, room - held)
        want_seqs += [s] * kept + [-1] * (n - kept)
        want_pos += [*range(held, held + kept)] + [-1] * (n - kept)
        kept = min(n, 16 * f.room[i] - held)  # (the cache's own table has none of the new pages)
        f.k[i].append(held, k[row:row + kept].float().numpy())
        f.v[i].append(held, v[row:row + kept].float().numpy())
        row += n
    assert seqs.tolist() == want_seqs + [-1] * 5 and pos.tolist() == want_pos + [-1] * 5
    if slots:
        assert ((at < 0) == (seqs < 0)).all()
    if grown:
        return
    f.cache.append_dev(0, k.cuda(), v.cuda(), seqs, pos, total + 5, stream())
    f.cache.check()
    f.check_rows()


@pytest.mark.gpu
@pytest.mark.parametrize("n,high,long,page", [(3, 40, 30, 16), (64, 300, 9, 16), (700, 100, 20, 48), (2500, 50, 60, 32)])
@pytest.mark.parametrize("room", [1, 0.37, 0.98])
def test_plan_of_more_rows_than_there_is_room_for(cuda_device, n, high, long, page, room):
    """Dropped rows are rows that were not brought: lengths, pages and growth agree with the rows that are left."""
    rng = np.random.default_rng(n)
    held, new = rng.integers(0, high + 1, n), rng.integers(0, long + 1, n)
    rows = room if isinstance(room, int) else int(new.sum() * room)
    front = np.concatenate([[0], np.cumsum(new)[:-1]])
    kept = np.clip(rows - front, 0, new)
    stride = max(1, int((-(-(held + kept) // page)).max()))  # (what is dropped need not fit the table)
    ids = rng.permutation(n + 3)[:n]
    table = rng.integers(0, 9999, (n + 3, stride)).astype(np.int32)
    free = rng.permutation(int((-(-(held + kept) // page) + -held // page).sum())).astype(np.int32)  # nor be paid in pages
    got, t = run_plan(ids, held, new, page, rows, free, table)
    want, w = plan_reference(ids.tolist(), held.tolist(), kept.tolist(), page, rows, free, table)
    want["status"][1] = 2
    for key, value in want.items():
        assert np.array_equal(got[key], value), key
    assert np.array_equal(t, w)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [5, 900])
def test_plan_without_row_arrays(cuda_device, n):
    """Nothing said about rows, no limit to them: lengths, starts and growth of the whole step."""
    rng = np.random.default_rng(n)
    held, new = rng.integers(0, 100, n), rng.integers(0, 40, n)
    table = np.full((n, 9), 5, np.int32)
    free = rng.permutation(int((-(-(held + new) // 16) + -held // 16).sum())).astype(np.int32)
    got, t = run_plan(range(n), held, new, 16, 0, free, table, skip=("row_seqs", "row_positions", "row_slots"))
    want, w = plan_reference(range(n), held.tolist(), new.tolist(), 16, int(new.sum()), free, table)
    for key in ("q_starts", "kv_lens", "page_starts", "status"):
        assert np.array_equal(got[key], want[key]), key
    assert np.array_equal(t, w)
    # room for none
    got, t = run_plan(range(n), held, new, 16, 1, free, table, skip=("row_positions", "row_slots"))
    assert got["status"].tolist()[1] == 2 and got["q_starts"][-1] == 1


@pytest.mark.gpu
def test_plan_with_a_table_that_is_only_read_flags_requests_outside_it(cuda_device):
    table = np.arange(40, dtype=np.int32).reshape(4, 10)
    got, t = run_plan([1, 3], [150, 20], [20, 3], 16, 24, None, table)
    assert got["status"].tolist() == [0, 8] and np.array_equal(t, table)
    assert got["row_slots"].tolist() == [19 * 16 + 6 + i for i in range(10)] + [-1] * 10 + [31 * 16 + 4 + i for i in range(3)] + [-1]
    assert got["row_seqs"].tolist() == [1] * 10 + [-1] * 10 + [3] * 3 + [-1]
    got, _ = run_plan([1, 3], [150, 20], [10, 3], 16, 24, None, table)  # to the row's end
    assert got["status"].tolist() == [0, 0]
    got, _ = run_plan([1, 9], [150, 20], [10, 3], 16, 24, None, table)
    assert got["status"].tolist() == [0, 8] and (got["row_seqs"][10:] == -1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,store", [("bf16", "i8"), ("f32", "f8")])
def test_steps_planned_on_the_gpu_and_replayed(cuda_device, dtype, store):
    """Plan, append and attention of a few steps, nothing read back in between; the last form captured once and replayed with other lengths."""
    n, nkvh, nh, d, most = 5, 2, 8, 64, 64
    f = Filled([0] * n, nkvh, d, dtype, store, extra=160)
    f.cache.flush()
    held = np.array([0, 0, 0, 0, 0])
    ids, q_starts, kv = i32(f.seqs), torch.empty(n + 1, dtype=torch.int32, device="cuda"), torch.empty(n, dtype=torch.int32, device="cuda")
    seqs, pos = (torch.empty(most, dtype=torch.int32, device="cuda") for _ in range(2))
    hd, nd = i32(held), i32(held)
    k, v = (torch.zeros(most, nkvh, d, dtype=TORCH[dtype], device="cuda") for _ in range(2))
    q, out = (torch.zeros(most, nh, d, dtype=TORCH[dtype], device="cuda") for _ in range(2))

    def step():
        llaisys.paged_plan_dev(stream=stream(), seq_ids_dev=ids, held_dev=hd, new_dev=nd, n_seqs=n, page_size=16, n_rows=most, q_starts_dev=q_starts,
                               kv_lens_dev=kv, row_seqs_dev=seqs, row_positions_dev=pos)
        f.cache.append_dev(0, k, v, seqs, pos, most, stream())
        f.cache.attention_dev(0, out, q, ids, q_starts, kv, n_seqs=n, total_q=most, max_q_len=most, max_kv_len=160, nh=nh, scale=d ** -0.5,
                              stream=stream())

    graph = None
    for turn, new in enumerate(([3, 20, 1, 0, 33], [1, 1, 1, 1, 1], [0, 17, 30, 5, 1], [1, 1, 0, 1, 1], [12, 0, 0, 40, 2])):
        new = np.array(new)
        total = int(new.sum())
        kr, vr, qr = f.rows(total), f.rows(total), torch.randn(total, nh, d).to(TORCH[dtype])
        for dst, src in ((k, kr), (v, vr), (q, qr)):
            dst[:total] = src.cuda()
        hd.copy_(i32(held))
        nd.copy_(i32(new))
        out.fill_(9.0)
        if turn < 2:
            step()
        else:
            if graph is None:
                graph = torch.cuda.CUDAGraph()
                torch.cuda.synchronize()
                with torch.cuda.graph(graph):
                    step()
            graph.replay()
        got, at = out.cpu().double(), 0
        assert (got[total:] == 9).all()
        for i in range(n):
            m = int(new[i])
            f.k[i].append(int(held[i]), kr[at:at + m].float().numpy())
            f.v[i].append(int(held[i]), vr[at:at + m].float().numpy())
            if m:
                kw, vw = (torch.from_numpy(x.worth()).double() for x in (f.k[i], f.v[i]))
                want, top, big = attention_f64(qr[at:at + m].double(), kw, vw, int(held[i]), d ** -0.5)
                assert ((got[at:at + m] - want).abs() <= tolerance(want, top, big, dtype, len(kw), d)).all()
            at += m
        held = held + new
    f.cache.check()
    f.check_rows()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,nh,d", [("bf16", 8, 128), ("f32", 4, 64)])
def test_steps_with_launch_overlap(cuda_device, dtype, nh, d):
    """Append and decode of every step launched under the kernels in front of them: the same bits, also behind calls in which nobody has a query."""
    n, steps = 37, 6
    rng = np.random.default_rng(2)
    lens = rng.integers(1, 300, n).tolist()
    most = max(lens) + steps
    outs = []
    for overlap in (False, True):
        f = Filled(lens, 2, d, dtype, "i8", extra=steps)
        f.cache.flush()
        torch.manual_seed(9)
        data = [tuple(torch.randn(n, h, d).to(TORCH[dtype]).cuda() for h in (2, 2, nh)) for _ in range(steps)]
        ids = i32(f.seqs)
        kv, pos = [i32([x + s + 1 for x in lens]) for s in range(steps)], [i32([x + s for x in lens]) for s in range(steps)]
        out = torch.zeros(steps, n, nh, d, dtype=TORCH[dtype], device="cuda")
        none = i32([0] * (n + 1))
        torch.cuda.synchronize()
        f.cache.set_launch_overlap(overlap)
        for s, (k, v, q) in enumerate(data):
            f.cache.append_dev(0, k, v, ids, pos[s], n, stream())
            f.cache.attention_dev(0, out[s], q, ids, none, kv[s], n_seqs=n, total_q=n, max_q_len=1, max_kv_len=most, nh=nh, scale=0.1, stream=stream())
            f.cache.decode_dev(0, out[s], q, ids, kv[s], n, most, nh, 0.1, stream())
        f.cache.check()
        outs.append(out.cpu())
    assert torch.equal(*outs) and outs[0].abs().max() > 0


@pytest.mark.gpu
def test_launch_overlap_of_two_caches(cuda_device):
    """Rows appended to a 16-bit cache, attention of an 8-bit one, decode of the first: with overlap the decode reads older pages ahead of its own wait,
    because the kernel in front of it was let go behind the append."""
    n, held, d, nh = 16, 2048, 128, 8
    f = Filled([300] * 8, 2, d, "bf16", "i8")
    pages = held // 16
    cache = llaisys.PagedKVCache(n * pages, 2, d, dtype=llaisys.DataType.BF16, device=llaisys.DeviceType.NVIDIA, max_seqs=n, max_pages_per_seq=pages)
    seqs = [cache.add_seq() for _ in range(n)]
    for i, s in enumerate(seqs):
        cache.assign_pages(s, range(i * pages, (i + 1) * pages))
    cache.flush()
    g = torch.Generator().manual_seed(1)
    rows = [[torch.randn(n * held, 2, d, generator=g).bfloat16().cuda() for _ in range(2)] for _ in range(3)]
    q8, q16 = torch.randn(8, nh, d, generator=g).bfloat16().cuda(), torch.randn(n, nh, d, generator=g).bfloat16().cuda()
    ids8, kv8, ids, kv = i32(f.seqs), i32([300] * 8), i32(seqs), i32([held] * n)
    seq, pos = i32(np.repeat(seqs, held)), i32(np.tile(np.arange(held), n))
    outs = []
    for overlap in (False, True):
        out8, out16 = (torch.zeros(3, *q.shape, dtype=q.dtype, device="cuda") for q in (q8, q16))
        torch.cuda.synchronize()
        cache.set_launch_overlap(overlap)
        f.cache.set_launch_overlap(overlap)
        for i, (k, v) in enumerate(rows):  # (the pages hold the turn before's rows until the append is through)
            cache.append_dev(0, k, v, seq, pos, n * held, stream())
            f.cache.decode_dev(0, out8[i], q8, ids8, kv8, 8, 300, nh, 0.1, stream())
            cache.decode_dev(0, out16[i], q16, ids, kv, n, held, nh, 0.1, stream())
        torch.cuda.synchronize()
        cache.check()
        f.cache.check()
        outs.append((out8.cpu(), out16.cpu()))
    for a, b in zip(*outs):
        assert torch.equal(a, b) and a.abs().max() > 0


@pytest.mark.gpu
def test_two_caches_on_two_streams_and_graphs(cuda_device):
    """Calls of two caches side by side, eager and replayed, give what they give alone."""
    sides = []
    for seed in (0, 1):
        f = Filled([700, 20, 333], 2, 128, "bf16", "i8", extra=4, seed=seed)
        f.cache.flush()
        q = torch.randn(600, 16, 128, generator=torch.Generator().manual_seed(seed)).bfloat16().cuda()
        sides.append((f, q, i32(f.seqs), i32([0, 400, 401, 600]), i32([700, 20, 333]), torch.cuda.Stream()))

    def call(side, chunk, dec):
        f, q, ids, starts, kv, _ = side
        f.cache.attention_dev(0, chunk, q, ids, starts, kv, n_seqs=3, total_q=600, max_q_len=400, max_kv_len=700, nh=16, scale=0.1, stream=stream())
        f.cache.decode_dev(0, dec, q, ids, kv, 3, 700, 16, 0.1, stream())

    def outputs():
        return [(torch.zeros_like(q), torch.zeros(3, 16, 128, dtype=q.dtype, device="cuda")) for _, q, *_ in sides]

    alone, eager, replayed = outputs(), outputs(), outputs()
    graphs = []
    for side, a in zip(sides, alone):
        call(side, *a)
    torch.cuda.synchronize()
    for side, r in zip(sides, replayed):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            call(side, *r)
    torch.cuda.synchronize()
    for _ in range(10):
        for side, e in zip(sides, eager):
            with torch.cuda.stream(side[5]):
                call(side, *e)
    torch.cuda.synchronize()
    for _ in range(10):
        for side, g in zip(sides, graphs):
            with torch.cuda.stream(side[5]):
                g.replay()
    torch.cuda.synchronize()
    for a, e, r in zip(alone, eager, replayed):
        for x, y, z in zip(a, e, r):
            assert torch.equal(x, y) and torch.equal(x, z)
    for f, *_ in sides:
        f.cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["decode", "pieces", "chunks"])
def test_waits_that_run_out_are_reported(cuda_device, form):
    """With a limit of a few polls the waits inside a healthy pipeline run out, from the first on or somewhere in the middle: the call ends, is reported,
    and the next one, with the limit as it was, gives the bits of the one before."""
    f = Filled([1700, 1, 45, 4300, 333], 2, 128, "bf16", "i8")
    counts = dict(decode=[1] * 5, pieces=[3, 1, 5, 2, 4], chunks=[700, 1, 40, 300, 333])[form]
    total = sum(counts)
    q = torch.randn(total, 12, 128, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    ids, starts, lens = i32(f.seqs), i32([0, *np.cumsum(counts).tolist()]), i32([1700, 1, 45, 4300, 333])
    out = torch.empty_like(q)

    def attend():
        out.fill_(torch.nan)
        f.cache.attention_dev(0, out, q, ids, None if form == "decode" else starts, lens, n_seqs=5, total_q=total, max_q_len=max(counts), max_kv_len=4300,
                              nh=12, scale=0.1, stream=stream())
        torch.cuda.synchronize()
        f.cache.check()
        return out.clone()

    first = attend()
    assert torch.isfinite(first).all()
    assert f.cache.last_kernel() == (llaisys.Kernel.EIGHT_BIT_TC if form == "chunks" else llaisys.Kernel.EIGHT_BIT)
    for polls in (0, 1, 2, 4, 8, 16, 64, 0):
        f.cache.set_wait_limit(polls)
        try:
            attend()
            assert polls > 0
        except llaisys.LlaisysError as e:
            assert e.status == Status.KERNEL
        f.cache.set_wait_limit(1 << 20)
        assert torch.equal(attend(), first), polls


@pytest.mark.gpu
@pytest.mark.parametrize("held,rows", [(2000, 900), (40, 40)])
def test_queries_end_with_the_call(cuda_device, held, rows):
    """q_starts that go on behind total_q: the queries there are none of the call's."""
    f = Filled([held], 2, 128, "bf16", "i8")
    q = torch.randn(rows, 8, 128).bfloat16().cuda()
    out, want = torch.full_like(q, 9.0), torch.empty(rows - 30, 8, 128, dtype=q.dtype, device="cuda")
    kw = dict(n_seqs=1, max_q_len=rows, nh=8, scale=0.1, stream=stream())
    f.cache.attention_dev(0, out, q, i32(f.seqs), i32([0, rows]), i32([held]), total_q=rows - 30, max_kv_len=held, **kw)
    f.cache.attention_dev(0, want, q, i32(f.seqs), i32([0, rows - 30]), i32([held]), total_q=rows - 30, max_kv_len=held, **kw)
    assert (out[rows - 30:] == 9).all() and torch.equal(out[:rows - 30], want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_gather_rows_of_a_plain_cache(cuda_device, dtype):
    cache = llaisys.PagedKVCache(9, 2, 64, dtype=NAMES[dtype], device=llaisys.DeviceType.NVIDIA, max_seqs=2)
    a, b = cache.add_seq(), cache.add_seq()
    cache.assign_pages(a, [7, 2])
    cache.assign_pages(b, [5])
    cache.flush()
    k, v = (torch.randn(40, 2, 64).to(TORCH[dtype]).cuda() for _ in range(2))
    seq, pos = [a] * 30 + [b] * 10, list(range(30)) + list(range(10))
    cache.append_dev(0, k, v, i32(seq), i32(pos), 40, stream())
    order = torch.randperm(40)
    out = [torch.zeros_like(k) for _ in range(2)]
    cache.gather_dev(0, *out, i32(seq)[order.cuda()].contiguous(), i32(pos)[order.cuda()].contiguous(), 40, stream())
    assert torch.equal(out[0], k[order.cuda()]) and torch.equal(out[1], v[order.cuda()])
    cache.check()


def test_gather_rows_of_a_cpu_cache():
    cache = llaisys.PagedKVCache(9, 2, 8, dtype=llaisys.DataType.F32, max_seqs=2)
    a = cache.add_seq()
    cache.assign_pages(a, [7, 2])
    k, v = torch.randn(20, 2, 8), torch.randn(20, 2, 8)
    cache.append(0, k, v, [a] * 20, range(20))
    out = [torch.full((3, 2, 8), 7.0) for _ in range(2)]
    seq, pos = np.array([a, 5, a], np.int32), np.array([17, 0, 3], np.int32)
    cache.gather_dev(0, *out, torch.from_numpy(seq), torch.from_numpy(pos), 3, None)
    assert torch.equal(out[0][0], k[17]) and torch.equal(out[1][2], v[3]) and (out[0][1] == 7).all()
    with pytest.raises(llaisys.LlaisysError):
        cache.check()


# ---- refusals --------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("changes,status", [(dict(store=llaisys.DataType.BF16), Status.INVALID), (dict(store=llaisys.DataType.U8), Status.INVALID),
                                            (dict(dtype=llaisys.DataType.I8), Status.INVALID), (dict(page_size=8), Status.INVALID),
                                            (dict(page_size=24), Status.INVALID), (dict(head_dim=80), Status.INVALID),
                                            (dict(head_dim=288), Status.INVALID), (dict(head_dim=0), Status.INVALID), (dict(nkvh=0), Status.INVALID),
                                            (dict(num_pages=0), Status.INVALID), (dict(device=llaisys.DeviceType.CPU), Status.UNSUPPORTED),
                                            (dict(device_id=99), Status.DEVICE)])
def test_refusals_of_the_cache(changes, status):
    with pytest.raises(llaisys.LlaisysError) as e:
        llaisys.PagedKVCache.quantized(**(dict(num_pages=4, nkvh=2, head_dim=64) | changes))
    assert e.value.status == status


@pytest.mark.parametrize("changes,status", [(dict(held_dev=0), Status.INVALID), (dict(new_dev=0), Status.INVALID), (dict(page_size=0), Status.INVALID),
                                            (dict(n_seqs=1 << 31), Status.INVALID), (dict(n_rows=1 << 31), Status.INVALID),
                                            (dict(n_free=1 << 40), Status.INVALID), (dict(row_slots_dev=64), Status.INVALID),
                                            (dict(free_pages_dev=64), Status.INVALID), (dict(table_stride=1 << 33), Status.INVALID)])
def test_refusals_of_the_plan(changes, status):
    args = LlaisysPagedPlan(**(dict(held_dev=64, new_dev=64, n_seqs=1, page_size=16, n_rows=1) | changes))
    assert LIB_LLAISYS.llaisysPagedPlanDev(int(llaisys.DeviceType.CPU), 0, ctypes.byref(args), None) == status
    assert LIB_LLAISYS.llaisysPagedPlanDev(int(llaisys.DeviceType.CPU), 0, None, None) == Status.INVALID
    args = LlaisysPagedPlan(held_dev=64, new_dev=64, n_seqs=1, page_size=16, n_rows=1)
    assert LIB_LLAISYS.llaisysPagedPlanDev(int(llaisys.DeviceType.CPU), 0, ctypes.byref(args), None) == Status.UNSUPPORTED


@pytest.mark.parametrize("changes", [dict(kv_lens_dev=4096), dict(q_starts_dev=4100), dict(row_positions_dev=4076), dict(status_dev=8188), dict(held_dev=4098),
                                     dict(row_slots_dev=65540, block_table_dev=1 << 20, table_rows=4, table_stride=4),
                                     dict(row_seqs_dev=(1 << 20) + 60, block_table_dev=1 << 20, table_rows=4, table_stride=4),
                                     dict(free_pages_dev=(1 << 20) + 60, n_free=1, block_table_dev=1 << 20, table_rows=4, table_stride=4)])
def test_refusals_of_a_plan_whose_arrays_overlap_or_are_not_aligned(changes):
    # (asked of a CPU, which has no such call: an argument that is not refused is never launched)
    args = LlaisysPagedPlan(**(dict(held_dev=4096, new_dev=8192, n_seqs=2, page_size=16, n_rows=7) | changes))
    assert LIB_LLAISYS.llaisysPagedPlanDev(int(llaisys.DeviceType.CPU), 0, ctypes.byref(args), None) == Status.INVALID


@pytest.mark.parametrize("changes", [dict(q_starts_dev=1 << 20, kv_lens_dev=1 << 20), dict(q_starts_dev=1 << 20, page_starts_dev=(1 << 20) + 8),
                                     dict(row_seqs_dev=1 << 20, row_positions_dev=(1 << 20) - 24), dict(status_dev=(1 << 20) + 52, row_slots_dev=1 << 20,
                                                                                                    block_table_dev=1 << 21, table_rows=4, table_stride=4)])
def test_refusals_of_a_plan_whose_outputs_lie_over_one_another(changes):
    args = LlaisysPagedPlan(**(dict(held_dev=4096, new_dev=8192, n_seqs=2, page_size=16, n_rows=7) | changes))
    assert LIB_LLAISYS.llaisysPagedPlanDev(int(llaisys.DeviceType.CPU), 0, ctypes.byref(args), None) == Status.INVALID


def test_arrays_of_a_plan_may_lie_side_by_side():
    args = LlaisysPagedPlan(held_dev=4096, new_dev=4104, n_seqs=2, page_size=16, n_rows=7, kv_lens_dev=4112, q_starts_dev=4084, status_dev=4120)
    assert LIB_LLAISYS.llaisysPagedPlanDev(int(llaisys.DeviceType.CPU), 0, ctypes.byref(args), None) == Status.UNSUPPORTED


def test_refusal_of_a_pool_beyond_64_bits():
    with pytest.raises(llaisys.LlaisysError) as e:
        llaisys.PagedKVCache.quantized(num_pages=2 ** 31 - 1, nkvh=65535, head_dim=256, page_size=2 ** 30, max_pages_per_seq=1)
    assert e.value.status == Status.INVALID


@pytest.mark.gpu
def test_refusals_of_calls_that_need_wide_pages(cuda_device):
    f = Filled([5], 2, 128, "bf16", "i8")
    x = torch.zeros(64, 8, 128, dtype=torch.bfloat16, device="cuda")
    one, zero = i32([1]), i32([0])
    calls = [lambda c: c.rope_append_dev(0, x, x, None, zero, zero, 1, 4, 1e4, stream()),
             lambda c: c.norm_append_dev(0, stream(), proj=x, row_stride=1024, q_at=0, k_at=512, v_at=768, gate_at=-1, q_out=x, seq_ids_dev=zero,
                                         positions_dev=zero, n_rows=1, nh=4),
             lambda c: c.decode_step_dev(0, x, x, x, x, zero, one, 1, 1, 4, 1.0, stream()),
             lambda c: c.decode_step_host(0, x.cpu(), x.cpu(), x.cpu(), x.cpu(), [0], [1], 4, 1.0),
             lambda c: c.fade_dev(0, x, x, zero, None, one, n_seqs=1, total_q=1, max_q_len=1, max_kv_len=1, nh=4, scale=1.0, stream=stream(), fade_a=x,
                                  fade_b=x),
             lambda c: c.latent_append_dev(0, stream(), proj=x, q_norm=x, kv_norm=x, q_latent=x, seq_ids_dev=zero, positions_dev=zero, rank=128, nh=4,
                                           n_rows=1),
             lambda c: c.latent_gather_dev(0, x, 128, zero, zero, one, 1, 1, stream()),
             lambda c: c.expanded_dev(stream(), q=x, k=x, k_shared=x, v=x, out=x, page_starts_dev=zero, q_starts_dev=zero, kv_lens_dev=one, nh=4, n_seqs=1),
             lambda c: c.gates_dev(0, x, x, zero, None, one, n_seqs=1, total_q=1, max_q_len=1, max_kv_len=1, nh=4, scale=1.0, stream=stream())]
    for call in calls:
        with pytest.raises(llaisys.LlaisysError) as e:
            call(f.cache)
        assert e.value.status == Status.UNSUPPORTED
    for call in (lambda c: c.append_dev(0, None, x, zero, zero, 1, stream()), lambda c: c.gather_dev(0, x, None, zero, zero, 1, stream()),
                 lambda c: c.gather_dev(1, x, x, zero, zero, 1, stream()), lambda c: c.decode_dev(0, x, x, zero, one, 1, 1, 5, 1.0, stream()),
                 lambda c: c.decode_dev(0, x, x, zero, one, 1, 1 << 20, 4, 1.0, stream())):
        with pytest.raises(llaisys.LlaisysError) as e:
            call(f.cache)
        assert e.value.status == Status.INVALID
    f.check_rows()
