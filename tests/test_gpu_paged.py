"""The paged KV cache (pollux_amd.paged) against float64: writing and reading back, attention of one token and of chunks.

Bars.  Writing is bit-exact against the same rounding steps in torch.  Attention per element, relative to max |V| of
the sequence: fp32 scores of 24-term products of rows of norm about sqrt 24 (the error of a score, 24 * 2^-24 * 24,
over sqrt 24, moves a probability by as much; twice for both operands' parts of 22 bits) stay within 64 * 2^-24 for
scores of a few units; sums of probabilities and values add a few 2^-24.  So 128 * 2^-24 * max|V|, and 1e-5 relative
over all (fp32 outputs); fp16 and bf16 outputs add half a step of their type, eps / 2 of the value.
"""

import ctypes
import math

import pytest
import torch

from pollux_amd import _lib
from pollux_amd.model import RMSNorm
from pollux_amd.paged import PagedBatch, PagedKV, paged_attention, paged_read, paged_write

pytestmark = pytest.mark.gpu

KV = [torch.int8, torch.float16, torch.float32]
INV127 = torch.tensor(1 / 127, dtype=torch.float32)


def _norm64(x, w, eps=1e-8):
    x = x.double()
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()


def _stored(x, kv_dtype):
    """What the cache holds for fp32 rows x [..., 24], as fp32."""
    if kv_dtype != torch.int8:
        return x.to(kv_dtype).float()
    a = x.abs().amax(-1, keepdim=True)
    live = a >= 2.0 ** -116
    codes = (x * torch.where(live, torch.full_like(a, 127.0) / a, 0.0)).round().clamp(-127, 127)
    out = codes * torch.where(live, a * INV127.to(x.device), 0.0)
    return torch.where(torch.isfinite(x).all(-1, keepdim=True), out, math.nan)


def _ln(dev, g):
    ln = RMSNorm(24).to(dev)
    with torch.no_grad():
        ln.weight.copy_(1 + 0.1 * torch.randn(24, generator=g, device=dev))
    return ln


def _setup(dev, kv_lens, q_lens, heads, page, kv_dtype, seed, fill=math.nan):
    """Pages (everything `fill` to begin with, pages in a shuffled order) and the batch."""
    g = torch.Generator(device=dev).manual_seed(seed)
    counts = [-(-n // page) for n in kv_lens]
    pages = sum(counts) + 2
    perm = torch.randperm(pages, generator=g, device=dev).tolist()
    tables = []
    for c in counts:
        tables.append([perm.pop() for _ in range(c)])
    kv = PagedKV.allocate(pages, heads, page, kv_dtype, dev)
    for t in (kv.k, kv.v):
        t.fill_(-77 if kv_dtype == torch.int8 else fill)
    if kv_dtype == torch.int8:
        kv.k_scale.fill_(fill)
        kv.v_scale.fill_(fill)
    return g, kv, tables, PagedBatch.build(tables, kv_lens, q_lens, dev)


def _fill(g, kv, tables, kv_lens, dev):
    """All positions of all sequences written; the fp32 rows [heads, n, 24] that the cache then stands for."""
    batch = PagedBatch.build(tables, kv_lens, kv_lens, dev)
    c = kv.heads * 24
    k, v = (torch.randn(sum(kv_lens), c, generator=g, device=dev) for _ in range(2))
    paged_write(k, v, kv, batch)
    keys, values, at = [], [], 0
    for n in kv_lens:
        for x, to in ((k, keys), (v, values)):
            to.append(_stored(x[at:at + n].view(n, kv.heads, 24), kv.k.dtype).transpose(0, 1))
        at += n
    return keys, values


def _reference(q, keys, values, kv_lens, q_lens, ln):
    """[tokens, heads * 24] in float64 on the CPU-safe path (float64 products)."""
    out, at = [], 0
    for k, v, n, t in zip(keys, values, kv_lens, q_lens):
        heads = k.shape[0]
        x = q[at:at + t].double().view(t, heads, 24)
        at += t
        if ln is not None:
            x = _norm64(x, ln.weight)
        s = x.transpose(0, 1).contiguous() @ k.double().transpose(1, 2).contiguous() / math.sqrt(24)
        pos = torch.arange(n - t, n, device=q.device)
        s = s.masked_fill(torch.arange(n, device=q.device) > pos[:, None], -math.inf)
        p = torch.softmax(s, -1)
        p = torch.where((pos >= 0)[:, None], p, 0.0)
        out.append((p @ v.double()).transpose(0, 1).reshape(t, heads * 24))
    return torch.cat(out)


def _check(got, ref, values, label):
    eps = 0.0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2
    top = max((v.abs().max().item() for v in values if v.numel()), default=0.0)
    err = (got.double() - ref).abs()
    rel = ((got.double() - ref).norm() / ref.norm().clamp(min=1e-30)).item()
    print(f"[paged] {label}: max {err.max().item():.2e} rel {rel:.2e}", flush=True)
    assert (err <= 128 * 2.0 ** -24 * top + eps * ref.abs()).all()
    assert rel <= 1e-5 + eps


@pytest.mark.parametrize("kv_dtype", KV)
@pytest.mark.parametrize("x_dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kv_lens,q_lens,heads,page", [
    ([1], [1], 1, 8), ([33, 1, 0, 16], [33, 1, 0, 3], 3, 16), ([100, 7, 64], [40, 7, 1], 17, 32),
    ([5, 300], [2, 300], 48, 64)])
def test_write_and_read_back(dev, kv_dtype, x_dtype, kv_lens, q_lens, heads, page):
    if kv_dtype == torch.int8 and heads == 17:
        page = 8
    g, kv, tables, _ = _setup(dev, [max(a, b) for a, b in zip(kv_lens, q_lens)], q_lens, heads, page, kv_dtype, 3)
    kv_lens = [n if n >= t or t == 3 else t for n, t in zip(kv_lens, q_lens)]
    kv_lens[2:3] = [max(kv_lens[2], q_lens[2])] if len(kv_lens) > 2 else []
    batch = PagedBatch.build(tables, kv_lens, q_lens, dev)
    ln = _ln(dev, g)
    n = sum(q_lens)
    big = torch.randn(n + 2, 3 * heads * 24, generator=g, device=dev).to(x_dtype)  # stacked: k and v are slices
    k, v = big[:, :heads * 24], big[:, heads * 24:2 * heads * 24]
    before = [t.clone() for t in (kv.k, kv.v)]
    paged_write(k, v, kv, batch, k_ln=ln)
    kn = _norm64(k[:n].view(n, heads, 24), ln.weight).float()
    want = [_stored(kn, kv_dtype).view(n, -1), _stored(v[:n].float().reshape(n, heads, 24), kv_dtype).view(n, -1)]
    got = paged_read(kv, batch)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    # slots of no token of the batch are as they were
    for t, old in zip((kv.k, kv.v), before):
        mask = torch.ones(t.shape[0], page, dtype=torch.bool, device=dev)
        for table, total, new in zip(tables, kv_lens, q_lens):
            for j in range(max(0, total - new), total):
                mask[table[j // page], j % page] = False
        keep = mask[:, None, :, None].expand_as(t)
        assert torch.equal(t[keep].nan_to_num(7.0) if t.is_floating_point() else t[keep],
                           old[keep].nan_to_num(7.0) if t.is_floating_point() else old[keep])


def test_int8_rows_of_every_size(dev):
    heads = 10
    g, kv, tables, batch = _setup(dev, [1], [1], heads, 8, torch.int8, 1)
    x = torch.randn(heads, 24, generator=g, device=dev)
    x[0] = 0.0
    x[1] *= 1e-37  # 127 / max|x| leaves fp32: zeros
    x[2] *= 1e-34
    x[3] *= 1e37
    x[4, 5] = math.inf
    x[5, 0] = math.nan
    x[6, 7] = -math.inf
    x[7] = 3.0  # every value the maximum
    x[8] = 1e-45  # the smallest fp32 number
    x[9, 3] = 3.4e38
    paged_write(x.view(1, -1), x.view(1, -1), kv, batch)
    got = paged_read(kv, batch)
    want = _stored(x, torch.int8).view(1, -1)
    for a in got:
        assert torch.equal(a.isnan(), want.isnan()) and torch.equal(a.nan_to_num(0.0), want.nan_to_num(0.0))
    assert (got[0].view(heads, 24)[[0, 1, 8]] == 0).all() and got[0].view(heads, 24)[[4, 5, 6]].isnan().all()


@pytest.mark.parametrize("kv_dtype", KV)
@pytest.mark.parametrize("kv_lens,heads,page", [
    ([1], 1, 8), ([2, 1, 3], 2, 8), ([63, 64, 65, 1], 3, 16), ([255, 256, 257], 2, 64), ([1023, 1024, 1025], 2, 128),
    ([777], 48, 64), ([0, 5], 2, 16), ([9001, 17], 2, 32), ([5000], 1, 4096)])
def test_one_token(dev, kv_dtype, kv_lens, heads, page):
    q_lens = [1] * len(kv_lens)
    g, kv, tables, batch = _setup(dev, kv_lens, q_lens, heads, page, kv_dtype, sum(kv_lens))
    keys, values = _fill(g, kv, tables, kv_lens, dev)
    q = torch.randn(len(kv_lens), heads * 24, generator=g, device=dev)
    ln = _ln(dev, g)
    _check(paged_attention(q, kv, batch, q_ln=ln), _reference(q, keys, values, kv_lens, q_lens, ln), values,
           f"one {kv_dtype} {kv_lens}")


@pytest.mark.parametrize("kv_dtype", KV)
def test_many_short_sequences(dev, kv_dtype):
    # 2,048 (sequence, head) pairs and more: a wave each
    kv_lens = [1 + 7 * i % 251 for i in range(65)]
    kv_lens[3] = 0
    q_lens, heads = [1] * 65, 33
    g, kv, tables, batch = _setup(dev, kv_lens, q_lens, heads, 16, kv_dtype, 77)
    keys, values = _fill(g, kv, tables, kv_lens, dev)
    q = torch.randn(65, heads * 24, generator=g, device=dev)
    ln = _ln(dev, g)
    _check(paged_attention(q, kv, batch, q_ln=ln), _reference(q, keys, values, kv_lens, q_lens, ln), values,
           f"many {kv_dtype}")


CHUNKS = [
    ([2], [2], 1, 8), ([31, 32, 33], [31, 32, 33], 2, 16), ([64, 65, 63], [64, 65, 63], 2, 64),
    ([127, 128, 129], [127, 128, 129], 3, 32), ([300, 70], [5, 70], 3, 16), ([1, 2, 500], [1, 2, 40], 2, 16),
    ([700, 33, 900, 5], [130, 1, 1, 5], 3, 32), ([257], [257], 1, 4096), ([3, 0, 64], [7, 0, 64], 2, 8),
    ([5000, 40], [33, 3], 2, 64), ([2500], [200], 1, 16)]


@pytest.mark.parametrize("kv_dtype", KV)
@pytest.mark.parametrize("kv_lens,q_lens,heads,page", CHUNKS)
def test_chunks(dev, kv_dtype, kv_lens, q_lens, heads, page):
    g, kv, tables, batch = _setup(dev, kv_lens, q_lens, heads, page, kv_dtype, sum(kv_lens))
    keys, values = _fill(g, kv, tables, kv_lens, dev)
    q = torch.randn(sum(q_lens), heads * 24, generator=g, device=dev)
    ln = _ln(dev, g)
    got = paged_attention(q, kv, batch, q_ln=ln)
    _check(got, _reference(q, keys, values, kv_lens, q_lens, ln), values, f"chunk {kv_dtype} {kv_lens} {q_lens}")
    # the same through the chunk kernel alone: no hint of one-token sequences
    plain = PagedBatch(batch.table, batch.cu_q, batch.kv_len, batch.tokens, batch.max_q, batch.max_kv)
    _check(paged_attention(q, kv, plain, q_ln=ln), _reference(q, keys, values, kv_lens, q_lens, ln), values, "no hint")


@pytest.mark.parametrize("kv_dtype", KV)
@pytest.mark.parametrize("x_dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("q_lens", [[1, 1], [40, 1]])
def test_16_bit_activations(dev, kv_dtype, x_dtype, q_lens):
    kv_lens, heads = [300, 77], 5
    g, kv, tables, batch = _setup(dev, kv_lens, q_lens, heads, 16, kv_dtype, 9)
    keys, values = _fill(g, kv, tables, kv_lens, dev)
    q = torch.randn(sum(q_lens), heads * 24, generator=g, device=dev).to(x_dtype)
    _check(paged_attention(q, kv, batch), _reference(q, keys, values, kv_lens, q_lens, None), values, f"{x_dtype}")


def test_strides_padding_rows_and_out(dev):
    kv_lens, q_lens, heads = [40, 9], [12, 9], 3
    g, kv, tables, batch = _setup(dev, kv_lens, q_lens, heads, 16, torch.int8, 4)
    keys, values = _fill(g, kv, tables, kv_lens, dev)
    stack = torch.randn(1, 30, 9 * 24, generator=g, device=dev)  # 30 rows, 21 of them the batch's
    q = stack[:, :, 3 * 24:6 * 24]
    ref = _reference(q[0], keys, values, kv_lens, q_lens, None)
    out = torch.full((1, 30, 72), 5.0, device=dev)
    assert paged_attention(q, kv, batch, out=out) is out
    _check(out[0, :21], ref, values, "slice")
    assert (out[0, 21:] == 5.0).all()
    assert (paged_attention(q, kv, batch)[0, 21:] == 0).all()
    odd = torch.empty(21 * 73 + 1, device=dev)[1:].view(21, 73)[:, :72]  # rows of no 16-byte alignment
    odd.copy_(q[0, :21])
    _check(paged_attention(odd, kv, batch), ref, values, "odd rows")
    kv2 = PagedKV.allocate(kv.k.shape[0], heads, 16, torch.int8, dev)
    paged_write(odd, odd, kv2, batch)
    assert torch.equal(paged_read(kv2, batch)[0], _stored(odd.reshape(21, 3, 24), torch.int8).view(21, -1))


@pytest.mark.parametrize("kv_dtype", KV)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("row", [0, 63, 70, 200])
def test_a_bad_row_reaches_no_earlier_token(dev, kv_dtype, bad, row):
    kv_lens, q_lens, heads = [260, 90], [200, 90], 2
    g, kv, tables, batch = _setup(dev, kv_lens, q_lens, heads, 32, kv_dtype, 12)
    _fill(g, kv, tables, kv_lens, dev)
    q = torch.randn(290, heads * 24, generator=g, device=dev)
    ref = paged_attention(q, kv, batch)
    one = PagedBatch.build([tables[0]], [row + 1], [1], dev)  # rewrite that token of the first sequence
    k, v = paged_read(kv, one)
    v[0, 3] = bad
    k[0, 30] = bad
    paged_write(k, v, kv, one)
    got = paged_attention(q, kv, batch)
    tol = 128 * 2.0 ** -24 * 6.0  # (values of unit variance: none past 6)
    first = max(0, row - 60)  # the first query (position 60 + i) at or after the row
    assert ((got[:first] - ref[:first]).abs() <= tol).all() and ((got[200:] - ref[200:]).abs() <= tol).all()
    assert not torch.isfinite(got[first:200, 3]).any()
    # head 1: a score of NaN or +inf makes the softmax NaN, one of -inf (the query's sign) leaves the key out
    keys, _ = paged_read(kv, PagedBatch.build([tables[0]], [260], [260], dev))
    ref = _reference(q[:200, 24:], [keys[:, None, 24:].transpose(0, 1)], [torch.ones(1, 260, 24, device=dev)], [260],
                     [200], None)
    want = ref[first:].isnan()
    assert want.any() and torch.equal(torch.isnan(got[first:200, 24:]), want)
    single = PagedBatch.build([tables[0]], [260], [1], dev)
    assert torch.equal(torch.isnan(paged_attention(q[199:200], kv, single)[0, 24:]), ref[199].isnan())


@pytest.mark.parametrize("size", [1e-12, 30.0, 1e4, 1e9])
@pytest.mark.parametrize("kv_dtype", [torch.int8, torch.float32])
def test_scores_of_any_size(dev, kv_dtype, size):
    # where one key's score leads by more than the roundings of the scores (48 * 2^-24 of the products' sizes) and 40,
    # the output is its value
    kv_lens, q_lens, heads = [400, 300], [200, 1], 3
    g, kv, tables, batch = _setup(dev, kv_lens, q_lens, heads, 16, kv_dtype, 8)
    full = PagedBatch.build(tables, kv_lens, kv_lens, dev)
    ln = _ln(dev, g)
    with torch.no_grad():
        ln.weight.mul_(size)
    k, v = (torch.randn(700, heads * 24, generator=g, device=dev) for _ in range(2))
    paged_write(k, v, kv, full, k_ln=ln)
    k, v = (x.view(700, heads, 24) for x in paged_read(kv, full))
    q = torch.randn(201, heads * 24, generator=g, device=dev)
    got = paged_attention(q, kv, batch, q_ln=ln).view(201, heads, 24)
    assert torch.isfinite(got).all()
    if size < 1:  # scores of nothing: the mean of the values seen
        want = v[:400].double().cumsum(0)[200:] / torch.arange(201, 401, device=dev)[:, None, None]
        assert ((got[:200] - want).abs() <= 128 * 2.0 ** -24 * v.abs().max()).all()
        return
    qn = _norm64(q.view(201, heads, 24), ln.weight)
    checked = 0
    for rows, keys, values in ((slice(0, 200), k[:400], v[:400]), (slice(200, 201), k[400:], v[400:])):
        x, kk = qn[rows].transpose(0, 1).contiguous(), keys.double().permute(1, 2, 0).contiguous()
        s = x @ kk / math.sqrt(24)
        unsure = 48 * 2.0 ** -24 * (x.abs() @ kk.abs()).amax(-1) / math.sqrt(24)
        n, t = keys.shape[0], x.shape[1]
        s = s.masked_fill(torch.arange(n, device=dev) > torch.arange(n - t, n, device=dev)[:, None], -math.inf)
        top = s.topk(2, -1)
        lead = top.values[..., 0] - top.values[..., 1] > 2 * unsure + 40
        want = values.transpose(0, 1)[torch.arange(heads, device=dev)[:, None], top.indices[..., 0]]
        o = got[rows].transpose(0, 1)
        assert ((o - want)[lead].abs() <= 4e-6 * values.abs().max()).all()
        checked += int(lead.sum())
    assert checked > (100 if size > 100 else 0)


def test_values_of_any_size(dev):
    # fp32 and int8 values over 60 orders of magnitude between tokens: nothing leaves the parts' range
    for kv_dtype in (torch.float32, torch.int8):
        kv_lens, q_lens, heads = [513], [300], 2
        g, kv, tables, batch = _setup(dev, kv_lens, q_lens, heads, 64, kv_dtype, 6)
        full = PagedBatch.build(tables, kv_lens, kv_lens, dev)
        k, v = (torch.randn(513, heads * 24, generator=g, device=dev) for _ in range(2))
        v *= 10.0 ** torch.linspace(-30, 30, 513, device=dev)[:, None]  # later tokens ever larger
        paged_write(k, v, kv, full)
        keys, values = (x.view(513, heads, 24).transpose(0, 1) for x in paged_read(kv, full))
        q = torch.randn(300, heads * 24, generator=g, device=dev)
        got = paged_attention(q, kv, batch).double().view(300, heads, 24)
        ref = _reference(q, [keys], [values], kv_lens, q_lens, None).view(300, heads, 24)
        top = values.abs().amax(-1).cummax(-1).values[:, 213:].transpose(0, 1)  # the largest value each token sees
        assert ((got - ref).abs() <= 128 * 2.0 ** -24 * top[..., None].double()).all()


def test_any_order_of_the_sequences(dev):
    kv_lens, q_lens, heads = [70, 300, 5, 41, 200], [1, 150, 1, 41, 1], 3
    g, kv, tables, batch = _setup(dev, kv_lens, q_lens, heads, 16, torch.int8, 31)
    keys, values = _fill(g, kv, tables, kv_lens, dev)
    q = torch.randn(sum(q_lens), heads * 24, generator=g, device=dev)
    ref = _reference(q, keys, values, kv_lens, q_lens, None)
    assert batch.singles == 3 and sorted(batch.order.tolist()) == [0, 1, 2, 3, 4] and batch.order.tolist()[:2] == [1, 3]
    for order, singles in (([3, 1, 2, 0, 4], 3), ([1, 3, 4, 2, 0], 2), ([4, 0, 2, 1, 3], 0), ([0, 1, 2, 3, 4], 1)):
        b = PagedBatch(batch.table, batch.cu_q, batch.kv_len, batch.tokens, batch.max_q, batch.max_kv, singles,
                       torch.tensor(order, dtype=torch.int32, device=dev))
        _check(paged_attention(q, kv, b), ref, values, f"order {order} {singles}")
    # places that name no sequence are passed over
    b = PagedBatch(batch.table, batch.cu_q, batch.kv_len, batch.tokens, batch.max_q, batch.max_kv, 0,
                   torch.tensor([4, 0, 2, 1, 3], dtype=torch.int32, device=dev) + torch.tensor([0, 0, 0, 9, -9], device=dev,
                                                                                            dtype=torch.int32))
    out = paged_attention(q, kv, b, out=torch.full_like(q, 9.0))
    assert (out[1:151] == 9.0).all() and (out[152:193] == 9.0).all() and torch.isfinite(out).all()


@pytest.mark.parametrize("shape", ["rising", "falling", "saw", "one peak"])
@pytest.mark.parametrize("kv_dtype,q_len", [(torch.float32, 1), (torch.float32, 20), (torch.float32, 60),
                                            (torch.float16, 100), (torch.int8, 300), (torch.float32, 300)])
def test_scores_that_rise_along_the_keys(dev, kv_dtype, q_len, shape):
    """Maxima that creep up, jump or fall from tile to tile, scores from 0 to 12.

    A score of 12 from 24 equal products: parts of 22 bits on both sides and 24 sums in fp32 move it by at most
    (2 * 2^-22 + 24 * 2^-24) * 12 = 384 * 2^-24, a probability by that much of itself, the quotient by twice.
    """
    n, heads = 1000, 2
    g, kv, tables, batch = _setup(dev, [n], [q_len], heads, 16, kv_dtype, 61)
    at = torch.arange(n, device=dev) / n
    s = {"rising": 12 * at, "falling": 12 - 12 * at, "saw": 12 * ((at * 7) % 1.0),
         "one peak": 12.0 * (torch.arange(n, device=dev) == 500)}[shape]
    everything = PagedBatch.build(tables, [n], [n], dev)
    k = (s / math.sqrt(24)).view(n, 1).expand(n, heads * 24).contiguous()
    v = torch.randn(n, heads * 24, generator=g, device=dev)
    paged_write(k, v, kv, everything)
    keys, values = ([_stored(x.view(n, heads, 24), kv_dtype).transpose(0, 1)] for x in (k, v))
    q = torch.ones(q_len, heads * 24, device=dev)
    got, ref = paged_attention(q, kv, batch), _reference(q, keys, values, [n], [q_len], None)
    err = (got.double() - ref).abs().max().item()
    print(f"[paged] {shape} {kv_dtype} {q_len}: max {err:.2e}", flush=True)
    assert err <= 768 * 2.0 ** -24 * values[0].abs().max().item()


@pytest.mark.parametrize("seqs,kv_len", [(3, 70), (3, 5000), (50, 70)])
def test_bad_places_at_the_end_of_an_order(dev, seqs, kv_len):
    """A sequence whose length leaves its bound, and one of two tokens, where single tokens belong: NaN, others whole."""
    heads, q_lens = 48, [40] + [1] * (seqs - 1)
    g, kv, tables, batch = _setup(dev, [kv_len] * seqs, q_lens, heads, 64, torch.int8, 41)
    _fill(g, kv, tables, [kv_len] * seqs, dev)
    q = torch.randn(sum(q_lens), heads * 24, generator=g, device=dev)
    ref = paged_attention(q, kv, batch)
    batch.kv_len[1] = kv_len + 1
    got = paged_attention(q, kv, batch)
    assert torch.isnan(got[40]).all() and torch.equal(got[:40], ref[:40]) and torch.equal(got[41:], ref[41:])
    batch.kv_len[1] = kv_len
    batch.cu_q[2] += 1  # sequence 1: rows 40 and 41, the next one none
    got = paged_attention(q, kv, batch)
    assert torch.isnan(got[40:42]).all() and torch.equal(got[:40], ref[:40]) and torch.equal(got[42:], ref[42:])


@pytest.mark.parametrize("q_lens", [[1, 1], [70, 40]])
@pytest.mark.parametrize("kv_dtype", KV)
def test_a_bad_query_is_its_own(dev, kv_dtype, q_lens):
    """The tile of such a query takes its scores key by key in fp32, whose roundings are not those of the two fp16
    parts: its other rows are then other bits, held to the same bar (each way's error is within it by itself)."""
    kv_lens, heads = [90, 40], 2
    g, kv, tables, batch = _setup(dev, kv_lens, q_lens, heads, 16, kv_dtype, 13)
    keys, values = _fill(g, kv, tables, kv_lens, dev)
    q = torch.randn(sum(q_lens), heads * 24, generator=g, device=dev)
    ref = _reference(q, keys, values, kv_lens, q_lens, None)
    q[0, 5] = math.nan
    got = paged_attention(q, kv, batch)
    assert torch.isnan(got[0, :24]).all()
    got[0, :24], ref[0, :24] = 0.0, 0.0
    _check(got, ref, values, f"a bad query {kv_dtype} {q_lens}")


def test_sequences_out_of_bounds(dev):
    heads = 2
    g, kv, tables, batch = _setup(dev, [100, 50, 20], [40, 1, 20], heads, 16, torch.int8, 2, fill=0.0)
    keys, values = _fill(g, kv, tables, [100, 50, 20], dev)
    q = torch.randn(61, heads * 24, generator=g, device=dev)
    ref = paged_attention(q, kv, batch)
    before = kv.k.clone(), kv.v_scale.clone()
    for change in ("page", "negative page", "length", "negative length"):
        table, kv_len = batch.table.clone(), batch.kv_len.clone()
        if change == "page":
            table[0, 1] = kv.k.shape[0]
        elif change == "negative page":
            table[0, 1] = -1
        else:
            kv_len[0] = 101 if change == "length" else -3
        bad = PagedBatch(table, batch.cu_q, kv_len, 61, 40, 100, 1)
        got = paged_attention(q, kv, bad)
        assert torch.isnan(got[:40]).all() and torch.equal(got[40:], ref[40:]), change
        k, v = paged_read(kv, bad)
        wrong = slice(0, 40) if "length" in change else slice(0, 0)  # (page 1 holds positions 16 .. 31: not these)
        assert torch.isnan(k[wrong]).all() and torch.isfinite(v[40:]).all()
        if "length" in change:
            paged_write(q * 3, q * 3, kv, PagedBatch(table, batch.cu_q, kv_len, 40, 40, 100, 0))
            assert torch.equal(kv.k, before[0]) and torch.equal(kv.v_scale, before[1])
    one = PagedBatch.build(tables[:1], [100], [1], dev)
    table = one.table.clone()
    table[0, 6] = 10_000
    assert torch.isnan(paged_attention(q[:1], kv, PagedBatch(table, one.cu_q, one.kv_len, 1, 1, 100))).all()
    last = PagedBatch(table, one.cu_q, one.kv_len, 1, 1, 100)
    paged_write(q[:1], q[:1], kv, last)
    assert torch.equal(kv.k, before[0]) and torch.isnan(paged_read(kv, last)[0]).all()
    long = torch.tensor([101], dtype=torch.int32, device=dev)
    assert torch.isnan(paged_attention(q[:1], kv, PagedBatch(one.table, one.cu_q, long, 1, 1, 100))).all()


def test_offsets_past_32_bits(dev):
    # a pool of over 2^32 bytes and 2^31 values: the last pages hold the sequence
    heads, page = 64, 64
    pages = (1 << 32) // (heads * page * 24) + 500
    kv = PagedKV(*(torch.empty(pages, heads, page, 24, dtype=torch.int8, device=dev) for _ in range(2)),
                 *(torch.empty(pages, heads, page, device=dev) for _ in range(2)))
    tables, g = [[pages - 1, 3, pages - 2]], torch.Generator(device=dev).manual_seed(1)
    keys, values = _fill(g, kv, tables, [150], dev)
    q = torch.randn(20, heads * 24, generator=g, device=dev)
    _check(paged_attention(q, kv, PagedBatch.build(tables, [150], [20], dev)),
           _reference(q, keys, values, [150], [20], None), values, "far chunk")
    _check(paged_attention(q[:1], kv, PagedBatch.build(tables, [150], [1], dev)),
           _reference(q[:1], keys, values, [150], [1], None), values, "far token")


def test_no_sequences_and_no_tokens(dev):
    kv = PagedKV.allocate(4, 2, 16, torch.int8, dev)
    for batch in (PagedBatch.build([], [], [], dev), PagedBatch.build([[1]], [10], [0], dev)):
        q = torch.empty(0, 48, device=dev)
        assert paged_attention(q, kv, batch).shape == (0, 48)
        paged_write(q, q, kv, batch)
        assert paged_read(kv, batch)[0].shape == (0, 48)


def test_a_captured_step_follows_its_tensors(dev):
    # one graph of write + attention, replayed as the sequences grow; every replay against an eager step
    kv_lens, heads = [30, 500, 64], 4
    g, kv, tables, _ = _setup(dev, [600] * 3, [1] * 3, heads, 32, torch.int8, 21)
    _fill(g, kv, tables, kv_lens, dev)
    table = PagedBatch.build(tables, [600] * 3, [1] * 3, dev).table
    cu, kv_len = torch.arange(4, dtype=torch.int32, device=dev), torch.tensor(kv_lens, dtype=torch.int32, device=dev)
    batch = PagedBatch(table, cu, kv_len, 3, 1, 600)
    x = torch.randn(3, 3 * heads * 24, generator=g, device=dev)
    ln = _ln(dev, g)

    def step():
        q, k, v = x.split(heads * 24, dim=1)
        paged_write(k, v, kv, batch, k_ln=ln)
        return paged_attention(q, kv, batch, q_ln=ln)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for rep in range(4):
        kv_len += 1
        x.copy_(torch.randn(x.shape, generator=g, device=dev))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step()), rep


def test_another_stream(dev):
    kv_lens, q_lens, heads = [3000, 10], [1, 1], 3
    g, kv, tables, batch = _setup(dev, kv_lens, q_lens, heads, 16, torch.int8, 5)
    _fill(g, kv, tables, kv_lens, dev)
    q = torch.randn(2, heads * 24, generator=g, device=dev)
    ref = paged_attention(q, kv, batch)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:  # two calls at once, a workspace each
        with torch.cuda.stream(s):
            outs.append(paged_attention(q, kv, batch))
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref) for o in outs)


@pytest.mark.parametrize("kv_dtype", KV)
@pytest.mark.parametrize("q_lens", [[40, 40], [1, 1], [40, 1]])
def test_a_page_list_that_ends_before_its_sequence(dev, kv_dtype, q_lens):
    """Beside a longer list: what lies past it is written nowhere and NaN, and page 0 is whose it is."""
    heads, page, kv_lens = 3, 16, [40, 40]
    tables = [[0, 1, 2], [3]]  # 40 positions, 16 positions
    g = torch.Generator(device=dev).manual_seed(19)
    kv = PagedKV.allocate(5, heads, page, kv_dtype, dev)
    for t in (kv.k, kv.v, kv.k_scale, kv.v_scale):
        if t is not None:
            t.zero_()
    keys, values = _fill(g, kv, [tables[0]], [40], dev)
    before = [t.clone() for t in (kv.k, kv.v)]
    n = sum(q_lens)
    batch = PagedBatch.build(tables, kv_lens, q_lens, dev)
    short = PagedBatch.build([tables[1]], kv_lens[1:], q_lens[1:], dev)  # (alone its list does not hold them)
    x = torch.randn(n, heads * 24, generator=g, device=dev)
    second = slice(q_lens[0], n)
    only = PagedBatch(batch.table[1:].contiguous(), torch.tensor([0, q_lens[1]], dtype=torch.int32, device=dev),
                      batch.kv_len[1:].clone(), q_lens[1], q_lens[1], 40)
    with pytest.raises(ValueError, match="does not hold"):
        paged_write(x[second], x[second], kv, short)
    paged_write(x[second], x[second], kv, only)
    for t, old in zip((kv.k, kv.v), before):
        assert torch.equal(t[[0, 1, 2, 4]], old[[0, 1, 2, 4]])
    held = 16 if q_lens[1] == 40 else 0  # new tokens that have a page
    for got, want in zip(paged_read(kv, only), (x[second], x[second])):
        assert torch.equal(got[:held], _stored(want[:held].reshape(-1, heads, 24), kv_dtype).view(held, heads * 24))
        assert torch.isnan(got[held:]).all()
    q = torch.randn(n, heads * 24, generator=g, device=dev)
    got = paged_attention(q, kv, batch)
    _check(got[:q_lens[0]], _reference(q[:q_lens[0]], keys, values, [40], q_lens[:1], None), values, "the longer list")
    assert torch.isfinite(got[second][:held]).all() and torch.isnan(got[second][held:]).all()


def _read_into(kv, batch, rows):
    """paged_read into outputs of `rows` rows that hold 5."""
    k, v = (torch.full((rows, kv.heads * 24), 5.0, device=kv.k.device) for _ in range(2))
    st = _lib.lib().plx_paged_read(ctypes.byref(kv._c), ctypes.byref(batch._c), k.data_ptr(), v.data_ptr(),
                                   _lib.stream_of(kv.k.device))
    _lib.check(st, "paged_read")
    return k, v


@pytest.mark.parametrize("kv_dtype", KV)
@pytest.mark.parametrize("ordered", [True, False])
@pytest.mark.parametrize("kv_len,bounds,new", [
    (70, [1, 1, 1], [1, 2, 0]), (70, [1, 1, 1], [0, 2, 1]), (5000, [1, 1, 1], [1, 2, 0]),  # one token's kernel
    (70, [40, 40, 3], [3, 79, 1]), (700, [150, 150, 150], [150, 299, 1]), (5000, [20, 20, 1], [0, 41, 0]),
    (70, [8, 1, 1], [0, 10, 0])])
def test_more_new_tokens_than_the_bound(dev, kv_dtype, ordered, kv_len, bounds, new):
    """All of such a sequence's rows are NaN, also those past max_q and the tiles that it takes; the others are whole."""
    heads, page = 17, 16
    g, kv, tables, batch = _setup(dev, [kv_len] * 3, bounds, heads, page, kv_dtype, 23, fill=0.0)
    keys, values = _fill(g, kv, tables, [kv_len] * 3, dev)
    if not ordered:
        batch = PagedBatch(batch.table, batch.cu_q, batch.kv_len, batch.tokens, batch.max_q, batch.max_kv, batch.singles)
    starts = torch.tensor([0, *new], device=dev).cumsum(0)
    assert int(starts[-1]) <= batch.tokens and new[1] > batch.max_q
    batch.cu_q.copy_(starts)
    a, b, n = starts[1:].tolist()
    q = torch.randn(batch.tokens, heads * 24, generator=g, device=dev)
    got = paged_attention(q, kv, batch, out=torch.full_like(q, 5.0))
    k, v = _read_into(kv, batch, batch.tokens)
    for t in (got, k, v):
        assert torch.isnan(t[a:b]).all() and (t[n:] == 5.0).all() and torch.isfinite(t[:a]).all()
    for at, count, i in ((0, a, 0), (b, n - b, 2)):
        if not count:
            continue
        ref = _reference(q[at:at + count], keys[i:i + 1], values[i:i + 1], [kv_len], [count], None)
        _check(got[at:at + count], ref, values, f"beside it {kv_dtype} {new}")
        assert torch.equal(k[at:at + count], keys[i][:, kv_len - count:].transpose(0, 1).reshape(count, -1))
    before = kv.k.clone(), kv.v.clone()
    x = torch.randn(batch.tokens, heads * 24, generator=g, device=dev)
    batch.cu_q.copy_(torch.tensor([0, 0, new[1], new[1]], device=dev))
    paged_write(x, x, kv, batch)
    assert torch.equal(kv.k, before[0]) and torch.equal(kv.v, before[1])


@pytest.mark.parametrize("kv_dtype", KV)
def test_tokens_before_the_first_position(dev, kv_dtype):
    """kv_len below the new tokens: those before position 0 are not written and read as zeros."""
    kv_lens, q_lens, heads, page = [3, 0, 20], [7, 2, 20], 3, 8
    g, kv, tables, batch = _setup(dev, kv_lens, q_lens, heads, page, kv_dtype, 29, fill=7.0)
    before = [t.clone() for t in (kv.k, kv.v, kv.k_scale, kv.v_scale) if t is not None]
    k, v = (torch.randn(29, heads * 24, generator=g, device=dev) for _ in range(2))
    paged_write(k, v, kv, batch)
    for got, x in zip(_read_into(kv, batch, 30), (k, v)):
        want = _stored(x.view(29, heads, 24), kv_dtype).view(29, -1)
        want[:4], want[7:9] = 0.0, 0.0
        assert torch.equal(got[:29], want) and (got[29] == 5.0).all()
    slots = torch.zeros(kv.k.shape[0], page, dtype=torch.bool, device=dev)
    for table, n in zip(tables, kv_lens):
        for j in range(n):
            slots[table[j // page], j % page] = True
    for t, old in zip((t for t in (kv.k, kv.v, kv.k_scale, kv.v_scale) if t is not None), before):
        keep = ~slots[:, None].expand(t.shape[:3])
        assert torch.equal(t[keep], old[keep])


@pytest.mark.parametrize("size", [2.0 ** 18, 1e12, 1e30])
@pytest.mark.parametrize("which", ["key", "value"])
@pytest.mark.parametrize("kv_dtype", [torch.int8, torch.float32])
@pytest.mark.parametrize("kv_len,q_len", [(20, 20), (60, 60), (120, 120), (300, 300), (3000, 40), (2500, 200)])
def test_a_large_row_reaches_no_earlier_token(dev, kv_dtype, kv_len, q_len, which, size):
    """A key or value far above the others, finite: the tokens before it keep the bar, relative to what they see."""
    heads, row = 2, kv_len - 6
    g, kv, tables, batch = _setup(dev, [kv_len], [q_len], heads, 16, kv_dtype, 71)
    keys, values = _fill(g, kv, tables, [kv_len], dev)
    q = torch.randn(q_len, heads * 24, generator=g, device=dev)
    ref = _reference(q, keys, values, [kv_len], [q_len], None)
    full = PagedBatch.build(tables, [kv_len], [kv_len], dev)
    k, v = paged_read(kv, full)
    (k if which == "key" else v)[row] *= size
    paged_write(k, v, kv, full)
    before = q_len - 6
    _check(paged_attention(q, kv, batch)[:before], ref[:before], [x[:, :row] for x in values], f"{which} {size:.0e}")


@pytest.mark.parametrize("size", [1e6, 1e12, 1e30])
@pytest.mark.parametrize("kv_dtype", [torch.int8, torch.float32])
@pytest.mark.parametrize("kv_len,q_len", [(90, 1), (90, 20), (90, 60), (200, 120), (400, 300), (3000, 40), (2500, 200)])
def test_a_large_row_of_no_weight(dev, kv_dtype, kv_len, q_len, size):
    """A key that every query's score is below -10^5 for, its value large: it adds e^-100000 of that, which is nothing,
    and the others' keys and values, in its tile and in later ones, keep the bar by themselves."""
    heads, row = 2, 17
    g, kv, tables, batch = _setup(dev, [kv_len], [q_len], heads, 16, kv_dtype, 73)
    _fill(g, kv, tables, [kv_len], dev)
    full = PagedBatch.build(tables, [kv_len], [kv_len], dev)
    k, v = paged_read(kv, full)
    k[row], v[row] = -min(size, 1e20), size
    paged_write(k, v, kv, full)
    keys, values = (x.view(kv_len, heads, 24).transpose(0, 1) for x in paged_read(kv, full))
    q = torch.randn(q_len, heads * 24, generator=g, device=dev).abs() + 0.1
    got = paged_attention(q, kv, batch)
    ref = _reference(q, [keys], [values], [kv_len], [q_len], None)
    first = max(0, row + 1 - (kv_len - q_len))
    others = values.clone()
    others[:, row] = 0.0
    _check(got[first:], ref[first:], [others], f"no weight {size:.0e}")


@pytest.mark.parametrize("kv_dtype", [torch.int8, torch.float32])
@pytest.mark.parametrize("kv_len,q_len", [(5000, 1), (5000, 33), (5000, 60), (2500, 200), (700, 300)])
def test_values_near_the_largest_fp32_numbers(dev, kv_dtype, kv_len, q_len):
    """Values up to 1e33 of one sign, whole and in key ranges: their sums of weights up to 1 stay below 3e38."""
    heads = 2
    g, kv, tables, batch = _setup(dev, [kv_len], [q_len], heads, 16, kv_dtype, 79)
    full = PagedBatch.build(tables, [kv_len], [kv_len], dev)
    k = torch.randn(kv_len, heads * 24, generator=g, device=dev)
    v = (0.1 + torch.rand(kv_len, heads * 24, generator=g, device=dev)) * 1e33
    paged_write(k, v, kv, full)
    keys, values = (x.view(kv_len, heads, 24).transpose(0, 1) for x in paged_read(kv, full))
    q = torch.randn(q_len, heads * 24, generator=g, device=dev)
    _check(paged_attention(q, kv, batch), _reference(q, [keys], [values], [kv_len], [q_len], None), [values], "1e33")


@pytest.mark.parametrize("size", [2.0 ** -17, 1e-9, 1e-25])
@pytest.mark.parametrize("kv_dtype", [torch.int8, torch.float32])
@pytest.mark.parametrize("kv_len,q_len", [(90, 1), (20, 20), (90, 60), (200, 120), (400, 300), (3000, 40), (2500, 200)])
def test_small_rows_among_others(dev, kv_dtype, kv_len, q_len, size):
    """Every 16th value is small.  Where all the weight is theirs (scores of 58 more) the others add e^-58 = 2^-83 of
    theirs, so the bar is relative to the small ones down to 2^-60; where the weights are even, to the others."""
    heads = 2
    g, kv, tables, batch = _setup(dev, [kv_len], [q_len], heads, 16, kv_dtype, 83)
    full = PagedBatch.build(tables, [kv_len], [kv_len], dev)
    small = (torch.arange(kv_len, device=dev) % 16 == 0)[:, None]
    v = torch.randn(kv_len, heads * 24, generator=g, device=dev)
    v = torch.where(small, v * size, v)
    noise = torch.randn(kv_len, heads * 24, generator=g, device=dev)
    for k, label in ((noise, "even"), (torch.where(small, 6.0, -6.0) + 0.1 * noise, "all of it")):
        paged_write(k, v, kv, full)
        keys, values = (x.view(kv_len, heads, 24).transpose(0, 1) for x in paged_read(kv, full))
        q = torch.ones(q_len, heads * 24, device=dev) if label == "all of it" else \
            torch.randn(q_len, heads * 24, generator=g, device=dev)
        ref = _reference(q, [keys], [values], [kv_len], [q_len], None)
        bar = values[:, small[:, 0]] if label == "all of it" and size >= 2.0 ** -60 else values
        err = (paged_attention(q, kv, batch).double() - ref).abs().max().item()
        print(f"[paged] small {size:.0e} {label}: {err:.2e}", flush=True)
        assert err <= 128 * 2.0 ** -24 * bar.abs().max().item()
    # keys that are small: their scores are nothing, beside others of a few units
    paged_write(torch.where(small, noise * size, noise), v, kv, full)
    keys, values = (x.view(kv_len, heads, 24).transpose(0, 1) for x in paged_read(kv, full))
    q = torch.randn(q_len, heads * 24, generator=g, device=dev)
    _check(paged_attention(q, kv, batch), _reference(q, [keys], [values], [kv_len], [q_len], None), [values], "small keys")
