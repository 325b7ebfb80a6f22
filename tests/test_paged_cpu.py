"""Paged key-value cache: operators on the CPU, their refusals, the bookkeeping, models that extend cached sequences."""
import pytest
import torch

from _paged import append_ref, attention_ref, make_cache

from incin_b200.cache import CacheFull, PagedCache
from incin_b200.ops import functional as F


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("theta", [None, 10000.0])
def test_append_and_attention_match_their_definitions(dtype, theta):
    hq, hkv, D, P = 6, 2, 16, 16
    lengths, offsets = [21, 0, 40, 16], _i32(0, 5, 5, 20, 36)
    k, v, table, lens = make_cache(lengths, hkv, P, D, dtype, "cpu")
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(38, (hq + 2 * hkv) * D, generator=g).to(dtype)   # two rows behind the last sequence
    k0, v0 = k.clone(), v.clone()
    q = F.kv_append(qkv, k, v, table, lens, offsets, n_heads=hq, theta=theta)
    ref, pos = append_ref(qkv.view(38, -1, D), lens, offsets, hq + hkv, theta)
    u = torch.finfo(dtype).eps / 2
    close = lambda a, b: bool(((a.double() - b).abs() <= u * b.abs() + 8 * 2.0 ** -24 * 6).all())
    assert close(q[:36], ref[:36, :hq]) and not q[36:].any()
    written = torch.zeros(k.shape[0], P, dtype=torch.bool)
    for r in range(36):
        s = int((offsets[1:] <= r).sum())
        page, slot = int(table[s, pos[r] // P]), int(pos[r] % P)
        written[page, slot] = True
        assert close(k[page, :, slot], ref[r, hq:hq + hkv]) and torch.equal(v[page, :, slot].double(), ref[r, hq + hkv:])
    for new, old in ((k, k0), (v, v0)):
        keep = ~written[:, None, :, None].expand_as(new)
        assert torch.equal(new[keep].nan_to_num(7.0), old[keep].nan_to_num(7.0))
    out = F.prompt_attention(q, k, v, table, lens, offsets)
    want, bound = attention_ref(q, k, v, table, lens, offsets, D ** -0.5)
    assert ((out.double() - want).abs() <= bound).all() and not out[36:].any()
    one = F.decode_attention(q[:4], k, v, table, lens, scale=0.3)
    want, bound = attention_ref(q[:4], k, v, table, lens, None, 0.3)
    assert ((one.double() - want).abs() <= bound).all() and not one[1].any()


def test_keys_behind_a_row_do_not_enter_it():
    """Infinities and NaN among a prompt's later tokens stay out of the earlier ones."""
    k, v, table, lens = make_cache([9], 1, 16, 16, torch.float32, "cpu")
    k[table[0, 0].long(), 0, 6] = float("nan")
    v[table[0, 0].long(), 0, 7] = float("inf")
    out = F.prompt_attention(torch.randn(9, 2, 16), k, v, table, lens, _i32(0, 9))
    assert torch.isfinite(out[:6]).all() and out[6:].isnan().all()


def test_refusals():
    k, v, table, lens = make_cache([20, 3], 2, 16, 16, torch.float32, "cpu", poison=False)
    q, off = torch.randn(5, 4, 16), _i32(0, 3, 5)
    ok = dict(k_pages=k, v_pages=v, table=table, lengths=lens, offsets=off)
    F.prompt_attention(q, **ok)
    for bad in (dict(table=table.long()), dict(lengths=lens[:1]), dict(offsets=off[:2]), dict(offsets=None), dict(v_pages=v[:, :1]),
                dict(k_pages=k.bfloat16()), dict(k_pages=k[:, :, :8], v_pages=v[:, :, :8]), dict(lengths=lens.float()),
                dict(table=table.t()[:2].contiguous().t()), dict(table=table[0])):
        with pytest.raises(ValueError):
            F.prompt_attention(q, **{**ok, **bad})
    for x in (q[:, :3], q[..., :8], q[0], q.double()):
        with pytest.raises(ValueError):
            F.prompt_attention(x, **ok)
    for scale in (float("nan"), -1.0):
        with pytest.raises(ValueError):
            F.prompt_attention(q, **ok, scale=scale)
    with pytest.raises(ValueError):
        F.decode_attention(q, k, v, table, lens)           # five rows, two sequences
    with pytest.raises(RuntimeError, match="no_grad"):
        F.prompt_attention(q.clone().requires_grad_(), **ok)
    with torch.no_grad():
        F.prompt_attention(q.clone().requires_grad_(), **ok)
    for t, n, o in ((table, _i32(20, 400), off), (table, _i32(20, -1), off), (table, lens, _i32(0, 3, 9)), (table, lens, _i32(0, 1, 5)),
                    (torch.full_like(table, 99), lens, off), (torch.full_like(table, -1), lens, off)):
        with pytest.raises(IndexError):
            F.prompt_attention(q, k, v, t, n, o)
        with pytest.raises(IndexError):
            F.kv_append(torch.randn(5, 8 * 16), k, v, t, n, o, n_heads=4)
    for kw in (dict(n_heads=3), dict(n_heads=4, theta=0.5), dict(n_heads=4, theta=float("nan"))):
        with pytest.raises(ValueError):
            F.kv_append(torch.randn(5, 8 * 16), k, v, table, lens, off, **kw)


def test_copy_pages():
    st = torch.randn(3, 2, 9, 2, 16, 16)
    old = st.clone()
    assert F.copy_pages(st, _i32(1, 1, 4, 8), _i32(0, 7, 4, 2)) is st
    want = old.clone()
    want[:, :, [0, 7, 2]] = old[:, :, [1, 1, 8]]
    assert torch.equal(st, want)
    for a, b in (((0, 9), (1, 2)), ((0, 1), (2, -1)), ((0, 1), (2, 2)), ((0, 1), (1, 5))):
        with pytest.raises(IndexError):
            F.copy_pages(st, _i32(*a), _i32(*b))
    assert torch.equal(st, want)
    for s, a, b in ((st.transpose(0, 1), _i32(0), _i32(1)), (st, _i32(0, 1), _i32(1)), (st, _i32(0).long(), _i32(1)),
                    (torch.zeros(4, 1, 1, 3), _i32(0), _i32(1)), (st[0, 0, 0], _i32(0), _i32(1))):
        with pytest.raises(ValueError):
            F.copy_pages(s, a, b)
    F.copy_pages(st, _i32(), _i32())


class Mirror:
    """A cache whose one-element tokens are written by hand and followed by plain lists."""

    def __init__(self, pages, size=16):
        self.cache = PagedCache(2, 1, 1, pages, page_size=size, dtype=torch.float64, device="cpu")
        self.cache.storage.fill_(-1.0)
        self.tokens = {}
        self.count = 0

    def extend(self, seqs, counts):
        batch = self.cache.extend(seqs, counts)
        P = self.cache.page_size
        for i, (s, n) in enumerate(zip(seqs, counts)):
            for pos in range(batch.starts[i], batch.starts[i] + n):
                self.count += 1
                self.tokens[s].append(self.count)
                self.cache.storage[:, :, batch.table[i, pos // P], 0, pos % P, 0] = float(self.count)

    def check(self):
        c = self.cache
        held = [0] * c.n_pages
        for s, want in self.tokens.items():
            pages = c.pages_of(s)
            assert c.length(s) == len(want) and len(pages) == -(-len(want) // c.page_size)
            for p in pages:
                held[p] += 1
            got = c.storage[:, :, pages, 0, :, 0].reshape(2, 2, -1)[..., :len(want)] if pages else torch.zeros(2, 2, 0, dtype=torch.float64)
            assert (got == torch.tensor(want, dtype=torch.float64)).all()
        assert held == c._refs and sorted(c._free) == [p for p in range(c.n_pages) if not held[p]]


@pytest.mark.parametrize("seed", range(6))
def test_bookkeeping_follows_plain_lists(seed):
    import random
    rng = random.Random(seed)
    m = Mirror(24)
    for _ in range(250):
        live = list(m.tokens)
        what = rng.choice(["new", "fork", "free", "truncate", "extend", "extend", "extend", "compact"])
        if what == "new" and len(live) < 8:
            m.tokens[m.cache.new()] = []
        elif what == "fork" and live and len(live) < 12:
            s = rng.choice(live)
            m.tokens[m.cache.fork(s)] = list(m.tokens[s])
        elif what == "free" and live:
            s = rng.choice(live)
            m.cache.free(s)
            del m.tokens[s]
        elif what == "truncate" and live:
            s = rng.choice(live)
            n = rng.randint(0, len(m.tokens[s]))
            m.cache.truncate(s, n)
            del m.tokens[s][n:]
        elif what == "extend" and live:
            seqs = rng.sample(live, rng.randint(1, len(live)))
            try:
                m.extend(seqs, [rng.choice([0, 1, 1, rng.randint(0, 40)]) for _ in seqs])
            except CacheFull:
                pass
        elif what == "compact":
            n = m.cache.compact()
            assert n == m.cache.n_pages - m.cache.free_pages == max([p + 1 for s in m.tokens for p in m.cache.pages_of(s)], default=0)
        m.check()


def test_a_forked_open_page_is_copied_once_per_writer():
    m = Mirror(8)
    a = m.cache.new()
    m.tokens[a] = []
    m.extend([a], [20])
    forks = [m.cache.fork(a) for _ in range(3)]
    for f in forks:
        m.tokens[f] = list(m.tokens[a])
    assert m.cache.free_pages == 6
    m.extend([a] + forks, [1] * 4)          # three copies of one open page; the last owner keeps it
    m.check()
    assert m.cache.free_pages == 3 and len({m.cache.pages_of(s)[1] for s in [a] + forks}) == 4


def test_cache_refusals():
    c = PagedCache(1, 1, 8, 3, device="cpu", page_size=16)
    a, b = c.new(), c.new()
    with pytest.raises(CacheFull):
        c.extend([a, b], [40, 16])
    assert c.length(a) == 0 and c.free_pages == 3
    for seqs, counts in (([a, a], [1, 1]), ([a], [-1]), ([], []), ([a], [1, 2])):
        with pytest.raises(ValueError):
            c.extend(seqs, counts)
    with pytest.raises(KeyError):
        c.extend([a, 77])
    c.extend([a], [17])
    with pytest.raises(ValueError):
        c.truncate(a, 18)
    c.free(a)
    with pytest.raises(KeyError):
        c.length(a)
    assert c.free_pages == 3
    for bad in (dict(page_size=8), dict(pages=0)):
        with pytest.raises(ValueError):
            PagedCache(**{**dict(n_layer=1, n_kv_head=1, head_dim=8, pages=3, device="cpu"), **bad})


@pytest.mark.parametrize("kind", ["llama", "gpt2"])
def test_extending_equals_scoring_the_whole_text(kind):
    """Prompt, one token at a time, a fork, a free and a compaction between them: fp32 logits of every step are those of the
    whole text (sums of a few hundred terms in another order)."""
    from incin_b200.models.gpt2 import GPT2, GPT2Config
    from incin_b200.models.llama import Llama, LlamaConfig
    model = Llama(LlamaConfig.tiny(), seed=1) if kind == "llama" else GPT2(GPT2Config.tiny(), seed=1)
    g = torch.Generator().manual_seed(2)
    tok = torch.randint(0, 500, (2, 60), generator=g)
    with torch.no_grad():
        full = model(tok)
    c = PagedCache.of(model, pages=20, page_size=16)
    a, b = c.new(), c.new()
    near = lambda got, want: bool(((got - want).abs() <= 2.0 ** -24 * 300 * (want.abs().amax() + 1)).all())
    out = model.extend(torch.cat([tok[0, :16], tok[1, :33]]), c, [a, b], [16, 33])
    assert near(out[0], full[0, 15]) and near(out[1], full[1, 32])
    f = c.fork(a)
    out = model.extend(torch.cat([tok[0, 16:17], tok[1, 33:34], tok[0, 16:17]]), c, [a, b, f])
    assert near(out[0], full[0, 16]) and near(out[1], full[1, 33]) and near(out[2], full[0, 16])
    c.free(a)
    c.compact()
    out = model.extend(torch.cat([tok[1, 34:50], tok[0, 17:18]]), c, [b, f], [16, 1])
    assert near(out[0], full[1, 49]) and near(out[1], full[0, 17])
    for tokens, seqs, counts in ((tok[0, :3], [b], [2]), (tok[0, :0], [b], [0]), (tok[0], [b], None), (tok[0, :300], [b], [300])):
        with pytest.raises(ValueError):
            model.extend(tokens, c, seqs, counts)
    assert c.length(b) == 50


def test_descriptor_matches_the_header():
    """The bytes that the front end packs are the C structure, field by field."""
    import struct
    from incin_b200.ffi import parse_headers
    from incin_b200.ops import paged
    fields = next(s.fields for s in parse_headers()[0] if s.name == "incin_paged_desc")
    letter = lambda t: "P" if t.endswith("*") else {"long long": "q", "int": "i", "float": "f"}[t]
    want = struct.Struct("@" + "".join(letter(t) for _, t, _ in fields))
    packer = paged._pack_desc.__self__
    values = list(range(1, len(fields) + 1))
    assert packer.size == want.size and packer.pack(*values) == want.pack(*values)
