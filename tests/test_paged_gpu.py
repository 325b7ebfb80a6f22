"""Paged key-value cache on the GPU: every operator against its definition in 64 bits, alone and as a model uses them."""
import threading

import pytest
import torch

from _paged import CONFIGS, append_ref, attention_ref, make_cache, tokens_of

pytestmark = pytest.mark.gpu


def _F():
    from incin_b200.ops import functional as F
    return F


def _status():
    from incin_b200.ops import gemm as G
    G.check_status()


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _randn(*shape, dtype, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def _same(a, b):
    """Equal bits, NaN included."""
    return torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))


# ------------------------------------------------------------------------------------------------------------- append
def _check_append(x2, hq, k, v, table, lens, offsets, theta):
    """Rows of the queries and slots of the cache after an append; nothing else may change."""
    F = _F()
    hkv, P, D = k.shape[1:]
    dtype = x2.dtype
    k0, v0 = k.clone(), v.clone()
    q = F.kv_append(x2, k, v, table, lens, offsets, n_heads=hq, theta=theta)
    _status()
    x = x2.reshape(x2.shape[0], hq + 2 * hkv, D)
    ref, pos = append_ref(x, lens.cpu(), None if offsets is None else offsets.cpu(), hq + hkv, theta)
    seq = torch.full((x.shape[0],), -1, dtype=torch.long)
    offs = list(range(x.shape[0] + 1)) if offsets is None else offsets.tolist()
    for s in range(len(offs) - 1):
        seq[offs[s]:offs[s + 1]] = s
    live = pos >= 0
    # one rounding (half a step); sine and cosine within 2^-22 (angle to 2^-24 of a turn), two products and a sum in fp32
    u = torch.finfo(dtype).eps / 2
    amp = x.double().cpu().view(*x.shape[:2], 2, D // 2).norm(dim=2).repeat(1, 1, 2)
    tol = u * ref.abs() + 2.0 ** -20 * amp + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    qd = q.double().cpu()
    assert ((qd - ref[:, :hq]).abs() <= tol[:, :hq])[live].all() and not qd[~live].any()
    page = table.cpu()[seq[live], pos[live] // P].long()
    slot = pos[live] % P
    kd = k.double().cpu()[page, :, slot]
    assert ((kd - ref[live, hq:hq + hkv]).abs() <= tol[live, hq:hq + hkv]).all()
    assert torch.equal(v.cpu()[page, :, slot], x[:, hq + hkv:].cpu()[live])
    if theta is None:
        assert torch.equal(q.cpu()[live], x[:, :hq].cpu()[live]) and torch.equal(k.cpu()[page, :, slot], x[:, hq:hq + hkv].cpu()[live])
    kept = torch.ones(k.shape[0], P, dtype=torch.bool)
    kept[page, slot] = False
    for new, old in ((k, k0), (v, v0)):
        new, old = (t.cpu().transpose(1, 2)[kept] for t in (new, old))
        assert _same(new, old)
    return q


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,D", CONFIGS)
@pytest.mark.parametrize("page,theta", [(16, 10000.0), (64, None), (128, 500000.0)])
def test_append_runs(dtype, hq, hkv, D, page, theta):
    """Runs of new tokens, none and one among them, behind cached ones; rows in front of nobody at the end."""
    new = [1, 0, 33, page, 17, 0]
    lengths = [1, 7, 40, page, 2 * page + 17, 0]
    k, v, table, lens = make_cache(lengths, hkv, page, D, dtype, "cuda", token_major=page == 64)
    offsets = _i32(0, *torch.tensor(new).cumsum(0).tolist())
    x = _randn(sum(new) + 3, (hq + 2 * hkv) * D, dtype=dtype, seed=page)
    _check_append(x, hq, k, v, table, lens, offsets, theta)


@pytest.mark.parametrize("rows", [1, 3, 700])
def test_append_one_token_each(rows):
    """One row per sequence, idle slots of the batch among them; rows of a wider buffer, 16-byte aligned or not."""
    hq, hkv, D = 4, 2, 64
    g = torch.Generator().manual_seed(rows)
    lengths = torch.randint(0, 70, (rows,), generator=g).tolist()
    for shift in (0, 8, 1):
        k, v, table, lens = make_cache(lengths, hkv, 16, D, torch.bfloat16, "cuda")
        wide = _randn(rows, (hq + 2 * hkv) * D + 24, dtype=torch.bfloat16)
        _check_append(wide[:, shift:shift + (hq + 2 * hkv) * D], hq, k, v, table, lens, None, 10000.0)


def test_append_far_positions():
    """A position of a million: the angle keeps its digits.  All entries in front of the new tokens name one shared page."""
    hq, hkv, D, P = 2, 1, 128, 64
    lengths, new = [1000003, 131072, 999], [40, 5, 999]
    width = max(lengths) // P + 1
    table = torch.zeros(3, width, dtype=torch.int32)
    at = 1
    for s, (n, t) in enumerate(zip(new, lengths)):
        for e in range((t - n) // P, (t - 1) // P + 1):
            table[s, e] = at
            at += 1
    k, v = (_randn(at, hkv, P, D, dtype=torch.float16, seed=s) for s in (1, 2))
    x = _randn(sum(new), (hq + 2 * hkv) * D, dtype=torch.float16, seed=3)
    _check_append(x, hq, k, v, table.cuda(), _i32(*lengths), _i32(0, 40, 45, 1044), 500000.0)


# ---------------------------------------------------------------------------------------------------------- attention
def _check_attention(q, k, v, table, lens, offsets=None, scale=None):
    F = _F()
    call = (lambda: F.decode_attention(q, k, v, table, lens, scale=scale)) if offsets is None else \
        (lambda: F.prompt_attention(q, k, v, table, lens, offsets, scale=scale))
    out = call()
    _status()
    ref, bound = attention_ref(q, k, v, table, lens, offsets, q.shape[-1] ** -0.5 if scale is None else scale)
    odd = ~torch.isfinite(ref)
    assert torch.equal(torch.isfinite(out), ~odd), "non-finite values in other places than the definition's"
    err = torch.where(odd, 0.0, (out.double() - ref).abs() - bound)
    assert (err <= 0).all(), f"worst excess {err.max().item():.3e}"
    assert _same(call(), out)      # sums have a fixed order
    return out


LENGTHS = [0, 1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 300, 1000]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,D", CONFIGS)
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_decode(dtype, hq, hkv, D, page):
    """Lengths around the tiles and page ends, an empty sequence, NaN in every slot that holds no token."""
    k, v, table, lens = make_cache(LENGTHS, hkv, page, D, dtype, "cuda", token_major=page == 32)
    _check_attention(_randn(len(LENGTHS), hq, D, dtype=dtype, seed=1), k, v, table, lens)


@pytest.mark.parametrize("lengths", [[1], [0], [5000], [33000, 1, 0, 700], [257] * 150, list(range(300)), [5] * 513 + [200] + [70] * 600])
@pytest.mark.parametrize("hq,hkv,D", [(32, 4, 64), (24, 8, 128), (2, 1, 128)])
def test_decode_balances_any_batch(lengths, hq, hkv, D):
    """One long sequence, one long among short ones, many equal ones, many different ones."""
    k, v, table, lens = make_cache(lengths, hkv, 64, D, torch.bfloat16, "cuda")
    _check_attention(_randn(len(lengths), hq, D, dtype=torch.bfloat16, seed=2), k, v, table, lens)


@pytest.mark.parametrize("what", ["decode", "prompt"])
@pytest.mark.parametrize("D", [64, 128])
def test_scores_that_grow_and_extreme_values(what, D):
    """The running maximum moves all along the keys; a key of infinite score, a NaN key, scores of -inf in front."""
    hq, hkv, n = 6, 2, 400
    k, v, table, lens = make_cache([n, n, n, n], hkv, 16, D, torch.bfloat16, "cuda")
    q = _randn(4, hq, D, dtype=torch.bfloat16, seed=3).abs() + 0.1
    for s in range(4):
        for j in range(n):
            page, slot = int(table[s, j // 16]), j % 16
            if s == 0:
                k[page, :, slot] *= 0.2 + 6.0 * j / n
            if s == 1 and j < 130:
                k[page, :, slot] = -float("inf")     # weight 0
            if s == 2 and j == 391:
                k[page, 0, slot] = float("nan")      # the first key head's queries only
            if s == 3 and j == 5:
                k[page, 1, slot] = float("inf")
    if what == "decode":
        out = _check_attention_values(q, k, v, table, lens, None)
    else:
        out = _check_attention_values(q.repeat_interleave(2, 0), k, v, table, lens, _i32(0, 2, 4, 6, 8))[::2]
    assert torch.isfinite(out[:2]).all()
    assert out[2, :3].isnan().all() and torch.isfinite(out[2, 3:]).all()
    assert out[3, 3:].isnan().all() and torch.isfinite(out[3, :3]).all()


def _check_attention_values(q, k, v, table, lens, offsets):
    """Finite rows against the definition; scores of -inf weigh 0 there too."""
    F = _F()
    out = F.decode_attention(q, k, v, table, lens) if offsets is None else F.prompt_attention(q, k, v, table, lens, offsets)
    _status()
    D = q.shape[-1]
    kk = k.clone()
    ninf = torch.isneginf(kk)
    kk[ninf] = -1e4      # a score below every other one by more than exp's range
    ref, bound = attention_ref(q, kk, v, table, lens, offsets, D ** -0.5)
    _, small = attention_ref(q, torch.where(ninf, 0.0, kk), v, table, lens, offsets, D ** -0.5)
    fine = torch.isfinite(ref).all(-1) & torch.isfinite(small).all(-1)
    assert ((out.double() - ref).abs() <= torch.minimum(bound, small * 1.5))[fine].all()
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,D", CONFIGS)
@pytest.mark.parametrize("page", [16, 64, 128])
def test_prompt(dtype, hq, hkv, D, page):
    """Runs of no, one and many new tokens without and behind cached ones; ends around the tiles; two rows behind the last."""
    new = [1, 0, 2, 17, 64, 129, 5, 200, 0]
    past = [0, 9, 31, 0, 64, 0, 300, 127, 0]
    lengths = [a + b for a, b in zip(new, past)]
    k, v, table, lens = make_cache(lengths, hkv, page, D, dtype, "cuda", token_major=page == 64)
    offsets = _i32(0, *torch.tensor(new).cumsum(0).tolist())
    q = _randn(sum(new) + 2, hq, D, dtype=dtype, seed=1)
    out = _check_attention(q, k, v, table, lens, offsets)
    assert not out[sum(new):].any()


@pytest.mark.parametrize("new,past", [([1], [0]), ([1], [7000]), ([3, 70], [9000, 0]), ([1500], [0]), ([1300, 1, 900], [0, 2000, 33]),
                                      ([1] * 40, list(range(40))), ([300] * 9, [0] * 9), ([31, 32, 33, 0, 257], [1000] * 5), ([0], [50])])
@pytest.mark.parametrize("hq,hkv,D", [(32, 4, 64), (24, 8, 128), (5, 5, 64), (16, 1, 128)])
def test_prompt_shapes(new, past, hq, hkv, D):
    """One row, a few rows over a long cache, long runs, many short ones."""
    lengths = [a + b for a, b in zip(new, past)]
    k, v, table, lens = make_cache(lengths, hkv, 32, D, torch.bfloat16, "cuda")
    offsets = _i32(0, *torch.tensor(new).cumsum(0).tolist())
    q = _randn(max(1, sum(new)), hq, D, dtype=torch.bfloat16, seed=len(new))
    _check_attention(q, k, v, table, lens, offsets)


@pytest.mark.parametrize("group", [3, 5, 7, 11, 12, 13, 15, 17, 24, 40])
@pytest.mark.parametrize("new,past", [([1, 9, 60], [0, 300, 0]), ([256], [5000]), ([333, 0, 1024], [0, 70, 129])])
@pytest.mark.parametrize("D", [64, 128])
def test_prompt_groups_across_tiles(group, new, past, D):
    """Groups that do not divide the rows of a query tile: tokens whose heads lie in two tiles, first and last rows of a run."""
    lengths = [a + b for a, b in zip(new, past)]
    k, v, table, lens = make_cache(lengths, 2, 16, D, torch.bfloat16, "cuda")
    q = _randn(sum(new), 2 * group, D, dtype=torch.bfloat16, seed=24)
    _check_attention(q, k, v, table, lens, _i32(0, *torch.tensor(new).cumsum(0).tolist()))


@pytest.mark.parametrize("hq,hkv,D", [(12, 12, 64), (32, 4, 64), (24, 8, 128)])
@pytest.mark.parametrize("at", [0, 5, 127, 128, 200, 299])
def test_prompt_later_tokens_stay_out(hq, hkv, D, at):
    """A NaN and an infinity among the values of one new token, a NaN in its key: earlier rows do not see them."""
    k, v, table, lens = make_cache([300, 450], hkv, 16, D, torch.bfloat16, "cuda")
    offsets = _i32(0, 300, 600)
    q = _randn(600, hq, D, dtype=torch.bfloat16, seed=4)
    page = table[:, at // 16].long()
    v[page[0], 0, at % 16, 3] = float("nan")
    v[page[0], 0, at % 16, 9] = float("inf")
    v[table[1, (150 + at) // 16].long(), 0, (150 + at) % 16, D - 1] = -float("inf")
    out = _check_attention(q, k, v, table, lens, offsets)
    assert torch.isfinite(out[:at]).all()
    v.nan_to_num_(0.0, 0.0, 0.0)
    k[page[0], 0, at % 16] = float("nan")
    out = _F().prompt_attention(q, k, v, table, lens, offsets)
    _status()
    group = hq // hkv
    assert torch.isfinite(out[:at]).all() and out[at:300, :group].isnan().all() and torch.isfinite(out[:, group:]).all()
    assert torch.isfinite(out[300:]).all()


@pytest.mark.parametrize("new,pad", [([1], 6000), ([700, 3], 4000), ([0, 0], 900), ([2000] * 3, 5000)])
def test_prompt_padded_batch(new, pad):
    """Many rows behind the last sequence, more than the work of the real ones: all of them zeros."""
    hq, hkv, D = 32, 4, 64
    k, v, table, lens = make_cache([max(n, 1) for n in new], hkv, 64, D, torch.bfloat16, "cuda")
    offsets = _i32(0, *torch.tensor(new).cumsum(0).tolist())
    q = _randn(sum(new) + pad, hq, D, dtype=torch.bfloat16, seed=9)
    for _ in range(5):
        torch.empty(q.shape, dtype=q.dtype, device="cuda").fill_(float("nan"))    # what the output's memory held before
        out = _F().prompt_attention(q, k, v, table, lens, offsets)
        assert not out[sum(new):].any()
    _check_attention(q, k, v, table, lens, offsets)


@pytest.mark.parametrize("hq,hkv,D", [(24, 8, 128), (32, 4, 64)])
@pytest.mark.parametrize("new,past", [([4], [32000]), ([100], [16000]), ([700, 900], [3000, 0])])
def test_prompt_repeats_to_the_bit(hq, hkv, D, new, past):
    """Calls in a row without waiting, over a cache larger than L2 among others: K and V tiles land out of order, calls overlap
    at their ends.  Sums have a fixed order, so any product that starts before its operands are complete shows up."""
    lengths = [a + b for a, b in zip(new, past)]
    offsets = _i32(0, *torch.tensor(new).cumsum(0).tolist())
    q = _randn(sum(new), hq, D, dtype=torch.bfloat16, seed=10)
    caches = [make_cache(lengths, hkv, 64, D, torch.bfloat16, "cuda", seed=s) for s in range(3)]
    first = [_F().prompt_attention(q, *c, offsets) for c in caches]
    _status()
    for _ in range(20):
        outs = [_F().prompt_attention(q, *c, offsets) for c in caches]
        for a, b in zip(outs, first):
            assert _same(a, b)
    _status()


def test_strided_queries_and_other_scales():
    hq, hkv, D = 8, 2, 64
    k, v, table, lens = make_cache([90, 40, 17], hkv, 32, D, torch.float16, "cuda")
    for shift in (0, 8, 3):
        flat = _randn(3, 4 * hq * D + 16, dtype=torch.float16, seed=5)
        q = flat[:, shift:shift + 2 * hq * D].view(3, 2 * hq, D)[:, ::2]
        _check_attention(q, k, v, table, lens, scale=0.0)
        _check_attention(q, k, v, table, lens, scale=0.31)
        _check_attention(q, k, v, table, lens, _i32(0, 1, 1, 3), scale=0.31)
        _check_attention(q.transpose(0, 1).contiguous().transpose(0, 1), k, v, table, lens, _i32(0, 0, 2, 3))
    wide = torch.cat([table, table, table], 1)[:, :table.shape[1]]     # rows of a wider table
    _check_attention(q, k, v, wide, lens)


@pytest.mark.parametrize("scale", [0.0, 1e-42, 1e-3, 2.0])
@pytest.mark.parametrize("D", [64, 128])
def test_scales(scale, D):
    """Scale 0, or one that 32 bits flush to 0, weighs all keys alike, those behind a row's last one not at all."""
    new, past = [200, 1, 0, 3], [100, 0, 7, 500]
    k, v, table, lens = make_cache([a + b for a, b in zip(new, past)], 2, 32, D, torch.bfloat16, "cuda")
    _check_attention(_randn(204, 6, D, dtype=torch.bfloat16), k, v, table, lens, _i32(0, 200, 201, 201, 204), scale=scale)
    _check_attention(_randn(4, 6, D, dtype=torch.bfloat16), k, v, table, lens, scale=scale)


@pytest.mark.parametrize("hq,hkv,D", [(128, 1, 64), (100, 1, 128), (66, 2, 64)])
def test_widest_groups(hq, hkv, D):
    """A query tile of one token; groups that fill it, or not."""
    new, past = [3, 1, 140], [0, 500, 60]
    lengths = [a + b for a, b in zip(new, past)]
    k, v, table, lens = make_cache(lengths, hkv, 16, D, torch.bfloat16, "cuda")
    q = _randn(144, hq, D, dtype=torch.bfloat16, seed=11)
    _check_attention(q, k, v, table, lens, _i32(0, 3, 4, 144))
    _check_attention(q[:3], k, v, table, lens)
    x = _randn(144, (hq + 2 * hkv) * D, dtype=torch.bfloat16, seed=12)
    _check_append(x, hq, k, v, table, lens, _i32(0, 3, 4, 144), 10000.0)


@pytest.mark.parametrize("hq,hkv,D", [(24, 8, 128), (32, 4, 64)])
@pytest.mark.parametrize("new,past", [([500], [0]), ([40, 3], [0, 900]), ([1, 0, 200], [0, 0, 5000])])
def test_wide_tables(hq, hkv, D, new, past):
    """Tables with room for far longer sequences, as a server keeps them for captured calls: entries behind the last token name
    no page; how far the keys are split changes on the device."""
    lengths = [a + b for a, b in zip(new, past)]
    k, v, table, lens = make_cache(lengths, hkv, 16, D, torch.bfloat16, "cuda")
    wide = torch.full((len(new), 8000), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    offsets = _i32(0, *torch.tensor(new).cumsum(0).tolist())
    _check_attention(_randn(sum(new) + 1, hq, D, dtype=torch.bfloat16, seed=15), k, v, wide, lens, offsets)
    _check_attention(_randn(len(new), hq, D, dtype=torch.bfloat16, seed=16), k, v, wide, lens)


def test_many_short_sequences():
    """More sequences than a warp, a launch or a table's rows hold at once; one table row for all of them."""
    hq, hkv, D = 8, 2, 64
    n = 1100
    k, v, table, _ = make_cache([90], hkv, 32, D, torch.bfloat16, "cuda")
    table = table.expand(n, -1)                       # rows that share their memory
    g = torch.Generator().manual_seed(1)
    lens = torch.randint(0, 91, (n,), generator=g).to(torch.int32).cuda()
    q = _randn(n, hq, D, dtype=torch.bfloat16, seed=13)
    _check_attention(q, k, v, table, lens)
    new = torch.minimum(torch.randint(0, 4, (n,), generator=g), lens.cpu())
    offsets = torch.cat([torch.zeros(1, dtype=torch.long), new.cumsum(0)]).to(torch.int32).cuda()
    rows = int(offsets[-1])
    _check_attention(_randn(rows, hq, D, dtype=torch.bfloat16, seed=14), k, v, table, lens, offsets)
    one = torch.tensor([[3, 9], [90, 9]], dtype=torch.int32, device="cuda")[:, 0]      # lengths with gaps: refused, one element is fine
    with pytest.raises(ValueError):
        _F().decode_attention(q[:2], k, v, table[:2], one)
    _check_attention(q[:1], k, v, table[:1], one[:1])


def test_odd_offsets_stay_in_bounds():
    """Offsets that fall, start late or pass the rows: every row is in bounds, rows that belong to one sequence are right."""
    F = _F()
    hq, hkv, D = 4, 2, 64
    lengths = [40, 50, 33]
    k, v, table, lens = make_cache(lengths, hkv, 16, D, torch.bfloat16, "cuda", poison=False)
    q = _randn(30, hq, D, dtype=torch.bfloat16)
    for offs in ((5, 10, 20, 30), (0, 10, 10, 500), (0, 25, 10, 30), (-7, 3, 2 ** 31 - 1, 4), (30, 20, 10, 0), (0, 0, 0, 0)):
        out = F.prompt_attention(q, k, v, table, lens, _i32(*offs))
        F.kv_append(_randn(30, (hq + 2 * hkv) * D, dtype=torch.bfloat16), k.clone(), v.clone(), table, lens, _i32(*offs), n_heads=hq)
        torch.cuda.synchronize()
        if offs == (5, 10, 20, 30):
            assert not out[:5].any()
            assert torch.equal(out[5:], F.prompt_attention(q[5:].clone(), k, v, table, lens, _i32(0, 5, 15, 25)))
    try:
        _status()
    except Exception:
        pass


def test_offsets_past_32_bits():
    """Pages whose elements lie beyond the first 2^31, keys and values in one tensor."""
    hq, hkv, D, P = 16, 8, 128, 128
    pages = 2 ** 31 // (hkv * P * D) + 40
    big = torch.empty(pages, hkv, P, D, dtype=torch.bfloat16, device="cuda")
    big[-40:].normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    table = torch.arange(pages - 40, pages, dtype=torch.int32, device="cuda").flip(0).view(2, 20)
    lens = _i32(2500, 1300)
    q = _randn(300, hq, D, dtype=torch.bfloat16, seed=6)
    _check_attention(q[:2], big, big, table, lens)
    _check_attention(q, big, big, table, lens, _i32(0, 200, 300))
    x = _randn(2, (hq + 2 * hkv) * D, dtype=torch.bfloat16, seed=7)
    _F().kv_append(x, big, big.clone(), table, lens, n_heads=hq)
    assert torch.equal(big[table[0, 2499 // P].long(), :, 2499 % P], x[0].view(-1, D)[hq:hq + hkv])
    _F().copy_pages(big[None], table[0, 3:4].contiguous(), _i32(5))
    assert torch.equal(big[5], big[table[0, 3].long()])
    _F().copy_pages(big[None], _i32(5), table[0, 4:5].contiguous())
    assert torch.equal(big[5], big[table[0, 4].long()])
    _status()


def test_bad_entries_are_reported_and_skipped():
    """Entries that name no page read as zeros and are not written through; other sequences are as ever."""
    from incin_b200 import _native as nat
    F = _F()
    hq, hkv, D, P = 4, 2, 64, 16
    lengths = [40, 50, 33]
    k, v, table, lens = make_cache(lengths, hkv, P, D, torch.bfloat16, "cuda")
    good = F.decode_attention(q := _randn(3, hq, D, dtype=torch.bfloat16), k, v, table, lens)
    for bad in (-1, k.shape[0], 2 ** 31 - 1, -2 ** 31):
        t = table.clone()
        t[1, 1] = bad
        out = F.decode_attention(q, k, v, t, lens)
        with pytest.raises(nat.NativeError):
            _status()
        zk, zv = k.clone(), v.clone()
        zk[table[1, 1].long()] = 0
        zv[table[1, 1].long()] = 0
        assert torch.equal(out[[0, 2]], good[[0, 2]]) and _same(out, F.decode_attention(q, zk, zv, table, lens))
        offsets = _i32(0, 1, 21, 22)
        qs = _randn(22, hq, D, dtype=torch.bfloat16, seed=8)
        out = F.prompt_attention(qs, k, v, t, lens, offsets)
        with pytest.raises(nat.NativeError):
            _status()
        assert _same(out, F.prompt_attention(qs, zk, zv, table, lens, offsets))
        k0, v0 = k.clone(), v.clone()
        t = table.clone()
        t[1, 3] = bad
        F.kv_append(_randn(3, (hq + 2 * hkv) * D, dtype=torch.bfloat16), k, v, t, lens, n_heads=hq)
        with pytest.raises(nat.NativeError):
            _status()
        changed = (k.view(torch.int16) != k0.view(torch.int16)).flatten(1).any(1)
        assert set(changed.nonzero().flatten().tolist()) <= {int(table[0, 2]), int(table[2, 2])}
        k.copy_(k0)
        v.copy_(v0)
    for n in (-5, 10 ** 6):
        F.decode_attention(q, k, v, table, _i32(40, n, 33))
        with pytest.raises(nat.NativeError):
            _status()
    F.kv_append(_randn(60, (hq + 2 * hkv) * D, dtype=torch.bfloat16), k, v, table, lens, _i32(0, 0, 60, 60), n_heads=hq)   # 60 rows, 50 tokens
    with pytest.raises(nat.NativeError):
        _status()


def test_cuda_refusals():
    from incin_b200 import _native as nat
    F = _F()
    for dtype, D in ((torch.float32, 64), (torch.bfloat16, 32), (torch.float16, 256)):
        k, v, table, lens = make_cache([20], 1, 16, D, dtype, "cuda", poison=False)
        q = torch.zeros(1, 2, D, dtype=dtype, device="cuda")
        for call in (lambda: F.decode_attention(q, k, v, table, lens), lambda: F.prompt_attention(q, k, v, table, lens, _i32(0, 1)),
                     lambda: F.kv_append(torch.zeros(1, 4 * D, dtype=dtype, device="cuda"), k, v, table, lens, n_heads=2)):
            with pytest.raises(nat.NativeError):
                call()
    k, v, table, lens = make_cache([20], 1, 16, 64, torch.bfloat16, "cuda")
    flat = torch.zeros(k.numel() + 8, dtype=torch.bfloat16, device="cuda")
    q = torch.zeros(1, 2, 64, dtype=torch.bfloat16, device="cuda")
    for bad in (flat[1:1 + k.numel()].view(k.shape), k.transpose(2, 3).contiguous().transpose(2, 3)):
        with pytest.raises(nat.NativeError):
            F.decode_attention(q, bad, v, table, lens)
    with pytest.raises(ValueError):
        F.decode_attention(q, k, v, table.cpu(), lens)
    with pytest.raises(nat.NativeError):
        F.decode_attention(torch.zeros(1, 129, 64, dtype=torch.bfloat16, device="cuda"), k, v, table, lens)
    with pytest.raises(RuntimeError):
        F.decode_attention(q.requires_grad_(), k, v, table, lens)


# -------------------------------------------------------------------------------------------------------------- pages
@pytest.mark.parametrize("lead,shape,pairs", [((), (9, 1, 16, 64), 3), ((3, 2), (9, 2, 16, 64), 1), ((22, 2), (70, 4, 64, 64), 30), ((2,), (4000, 1, 1, 8), 1900),
                                              ((1, 2), (40, 8, 128, 128), 17), ((5,), (7, 3, 5, 8), 2)])
def test_copy_pages(lead, shape, pairs):
    g = torch.Generator().manual_seed(pairs)
    st = _randn(*lead, *shape, dtype=torch.bfloat16)
    order = torch.randperm(shape[0], generator=g).to(torch.int32)
    src, dst = order[:pairs].clone(), order[pairs:2 * pairs].clone()
    src[-1] = src[0]                     # a page copied twice
    want = st.clone()
    want.view(-1, *shape)[:, dst.cuda().long()] = st.view(-1, *shape)[:, src.cuda().long()]
    assert _F().copy_pages(st, src.cuda(), dst.cuda()) is st
    _status()
    assert torch.equal(st, want)


def test_copy_pages_leaves_bad_pairs_out():
    from incin_b200 import _native as nat
    st = torch.arange(12, device="cuda", dtype=torch.float32).view(12, 1, 1, 1).expand(12, 1, 4, 4).contiguous()
    #        fine     twice: the first  bad pages              5 -> 6 -> 7: only 6 -> 7   itself
    src = _i32(0, 1, 2, 12, 3, -1, 5, 6, 8)
    dst = _i32(9, 10, 10, 11, 12, 4, 6, 7, 8)
    _F().copy_pages(st, src, dst)
    with pytest.raises(nat.NativeError):
        _status()
    assert st[:, 0, 0, 0].tolist() == [0, 1, 2, 3, 4, 5, 6, 6, 8, 0, 1, 11]


# ----------------------------------------------------------------------------------------------------------- together
def test_captured_step_follows_its_tables():
    """A captured append and attention, replayed while lengths and tables change; two captured graphs side by side on two
    streams; the results of eager calls to the bit."""
    F = _F()
    hq, hkv, D, P, S, W = 8, 2, 64, 16, 5, 40
    g = torch.Generator().manual_seed(0)
    sets = []
    for _ in range(2):
        k, v = (_randn(S * W, hkv, P, D, dtype=torch.bfloat16, seed=i) for i in (1, 2))
        table = torch.randperm(S * W, generator=g).to(torch.int32).view(S, W).cuda()
        x = _randn(S, (hq + 2 * hkv) * D, dtype=torch.bfloat16, seed=3)
        lens = torch.zeros(S, dtype=torch.int32, device="cuda")
        offs = torch.arange(S + 1, dtype=torch.int32, device="cuda")

        def step(x=x, k=k, v=v, table=table, lens=lens, offs=offs):
            q = F.kv_append(x, k, v, table, lens, n_heads=hq, theta=10000.0)
            return F.decode_attention(q, k, v, table, lens), F.prompt_attention(q, k, v, table, lens, offs)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                out = step()
        torch.cuda.current_stream().wait_stream(stream)
        sets.append((graph, stream, out, step, (x, table, lens)))
    for trial in range(6):
        for graph, stream, out, step, (x, table, lens) in sets:
            x.copy_(torch.randn(x.shape, generator=g).to(x.dtype))
            table.copy_(torch.randperm(S * W, generator=g).to(torch.int32).view(S, W))
            lens.copy_(torch.randint(0 if trial % 2 else 1, [W * P + 1, 2, 70][trial % 3], (S,), generator=g).to(torch.int32))
        torch.cuda.synchronize()
        for graph, stream, *_ in sets:
            with torch.cuda.stream(stream):
                for _ in range(3):
                    graph.replay()
        torch.cuda.synchronize()
        for graph, stream, out, step, (x, table, lens) in sets:
            want = step()
            idle = lens == 0
            assert _same(out[0], want[0]) and _same(out[1][~idle], want[1][~idle])
            assert not out[0][idle].any()
    try:
        _status()       # idle slots have a row each by the prompt's offsets, more rows than tokens
    except Exception:
        pass


def _two_batches():
    """Calls of decode and prompt attention over two caches, all with parts to join, and the results each gives alone."""
    F = _F()
    calls = []
    for seed, (hq, hkv, D) in enumerate([(24, 8, 128), (32, 4, 64)]):
        k, v, table, lens = make_cache([9000, 30, 0, 4000], hkv, 64, D, torch.bfloat16, "cuda", seed=seed)
        one, many = _randn(4, hq, D, dtype=torch.bfloat16, seed=seed), _randn(43, hq, D, dtype=torch.bfloat16, seed=seed + 2)
        offsets = _i32(0, 20, 23, 23, 43)
        calls.append(lambda a=(one, k, v, table, lens): F.decode_attention(*a))
        calls.append(lambda a=(many, k, v, table, lens, offsets): F.prompt_attention(*a))
    return calls, [c() for c in calls]


def test_streams_and_threads_side_by_side():
    calls, alone = _two_batches()
    torch.cuda.synchronize()
    results = [[] for _ in calls]

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(30):
                results[i].append(calls[i]())
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i, got in enumerate(results):
        assert len(got) == 30 and all(_same(x, alone[i]) for x in got)
    _status()


def test_captured_graphs_side_by_side():
    """Graphs of the same calls replayed at the same time on two streams have workspaces of their own."""
    calls, alone = _two_batches()
    graphs = []
    for order in (calls, calls[::-1]):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = [c() for c in order]
        graphs.append((graph, outs, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(10):
        for graph, _, stream in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for (_, outs, _), want in zip(graphs, (alone, alone[::-1])):
        assert all(_same(x, y) for x, y in zip(outs, want))
    _status()


@pytest.mark.parametrize("kind", ["llama", "gpt2"])
def test_model_extends_cached_sequences(kind):
    """Prompts of different lengths, a fork, single steps and a compaction in bf16 against the whole text in fp32."""
    import copy
    from incin_b200.cache import PagedCache
    from incin_b200.models.gpt2 import GPT2, GPT2Config
    from incin_b200.models.llama import Llama, LlamaConfig
    model = Llama(LlamaConfig.tiny(), seed=1) if kind == "llama" else GPT2(GPT2Config.tiny(), seed=1)
    tok = torch.randint(0, 500, (3, 100), generator=torch.Generator().manual_seed(2))
    with torch.no_grad():
        full = model(tok)
    gpu = copy.deepcopy(model).cuda().to(torch.bfloat16)
    c = PagedCache.of(gpu, pages=40, page_size=16)
    a, b, d = c.new(), c.new(), c.new()
    seen = []

    def ext(parts, seqs, counts=None):
        out = gpu.extend(torch.cat([tok[r, i:j] for r, i, j in parts]).cuda(), c, seqs, counts)
        seen.extend((o.float().cpu(), full[r, j - 1]) for o, (r, _, j) in zip(out, parts))
    ext([(0, 0, 64), (1, 0, 37), (2, 0, 1)], [a, b, d], [64, 37, 1])
    f = c.fork(b)
    ext([(0, 64, 65), (1, 37, 38), (2, 1, 2), (1, 37, 38)], [a, b, d, f])
    c.free(a)
    c.compact()
    ext([(1, 38, 90), (2, 2, 3), (1, 38, 39)], [b, d, f], [52, 1, 1])
    for i in range(39, 45):
        ext([(1, i, i + 1)], [f])
    _status()
    got, want = (torch.stack(t) for t in zip(*seen))
    # two layers in bf16: each of about eight roundings a layer adds half a step to every activation, 2^-8 sqrt(16) of the
    # logits' rms, four times that for the largest of a few thousand
    rms = want.pow(2).mean().sqrt()
    assert (got - want).abs().max() <= 16 * 2.0 ** -8 * rms * 2
    assert (got - want).pow(2).mean().sqrt() <= 4 * 2.0 ** -8 * rms


def test_model_matches_its_own_scoring_for_odd_batches():
    """Every split of one text into prompts and single steps ends in the same logits, up to bf16."""
    from incin_b200.cache import PagedCache
    from incin_b200.models.llama import Llama, LlamaConfig
    model = Llama(LlamaConfig.tiny(), seed=3).cuda().to(torch.bfloat16)
    tok = torch.randint(0, 500, (150,), generator=torch.Generator().manual_seed(4)).cuda()
    with torch.no_grad():
        want = model(tok[None])[0, -1].float()
    rms = want.pow(2).mean().sqrt()
    for cuts in ([150], [149, 1], [1, 149], [64, 64, 22], [127, 1, 1, 1, 20]):
        c = PagedCache.of(model, pages=8, page_size=32)
        s, at = c.new(), 0
        for n in cuts:
            out = model.extend(tok[at:at + n], c, [s], [n])
            at += n
        assert (out[0].float() - want).abs().max() <= 2 * 16 * 2.0 ** -8 * rms
    _status()
