"""Paged key-value cache on the CPU: steps that fail, and arguments at the edge of what the operators take."""
import pytest
import torch

from incin_b200.cache import PagedCache
from incin_b200.ops import functional as F
from incin_b200.ops import functional as F


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32)


def _model(kind):
    from incin_b200.models.gpt2 import GPT2, GPT2Config
    from incin_b200.models.llama import Llama, LlamaConfig
    return Llama(LlamaConfig.tiny(), seed=1) if kind == "llama" else GPT2(GPT2Config.tiny(), seed=1)


def _books(c, seqs):
    return [(c.length(s), c.pages_of(s)) for s in seqs], list(c._refs), sorted(c._free)


class Stop(BaseException):
    pass


@pytest.mark.parametrize("kind", ["llama", "gpt2"])
@pytest.mark.parametrize("where", ["token", "first layer", "last layer", "interrupt", "copy", "batch"])
def test_a_failed_step_is_taken_back(kind, where, monkeypatch):
    """Whatever raises inside a step, lengths, pages and their owners are as before, those of forked sequences too, and the next
    step gives the logits of the whole text."""
    import incin_b200.cache as cache_module
    model = _model(kind)
    tok = torch.randint(0, 500, (60,), generator=torch.Generator().manual_seed(2))
    with torch.no_grad():
        full = model(tok[None])[0]
    c = PagedCache.of(model, pages=12, page_size=16)
    a = c.new()
    model.extend(tok[:30], c, [a], [30])
    b = c.fork(a)                        # an open page of two owners
    before = _books(c, [a, b])

    def fail(*args, **kw):
        raise (Stop if where == "interrupt" else RuntimeError)("planted")
    for counts in ([1, 1], [20, 1], [2, 25]):
        tokens = torch.cat([tok[30:30 + n] for n in counts])
        with monkeypatch.context() as m:
            if where == "token":
                tokens[0] = 10 ** 6
            elif where == "copy":
                m.setattr(cache_module.F, "copy_pages", fail)
            elif where == "batch":
                m.setattr(cache_module.PagedBatch, "__init__", fail)
            else:
                m.setattr(model.blocks[0 if where == "first layer" else -1], "extend", fail)
            with pytest.raises(Stop if where == "interrupt" else (RuntimeError, IndexError)):
                model.extend(tokens, c, [a, b], counts)
        assert _books(c, [a, b]) == before
    out = model.extend(torch.cat([tok[30:37], tok[30:33]]), c, [a, b], [7, 3])
    # fp32 sums of a few hundred terms in another order
    for got, want in zip(out, (full[36], full[32])):
        assert (got - want).abs().max() <= 2.0 ** -24 * 300 * (want.abs().max() + 1)


def test_an_extension_can_be_taken_back():
    c = PagedCache(1, 1, 8, 6, device="cpu", page_size=16)
    a = c.new()
    c.extend([a], [20])
    b = c.fork(a)
    before = _books(c, [a, b])
    for counts in ([1, 1], [13, 0], [0, 30]):
        batch = c.extend([a, b], counts)
        assert _books(c, [a, b]) != before
        c.take_back(batch)
        assert _books(c, [a, b]) == before
        c.take_back(batch)               # once only
        assert _books(c, [a, b]) == before


def test_forward_mode_is_refused():
    """A tangent is refused like an input that wants a gradient, by every operator and for every floating input."""
    import torch.autograd.forward_ad as fw
    k, v = torch.randn(4, 2, 16, 16), torch.randn(4, 2, 16, 16)
    table, lens, off = _i32(0, 1, 2, 3).view(2, 2), _i32(20, 3), _i32(0, 1, 2)
    q, x = torch.randn(2, 4, 16), torch.randn(2, 8 * 16)
    want = F.decode_attention(q, k, v, table, lens)
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))
        calls = [lambda: F.decode_attention(dual(q), k, v, table, lens), lambda: F.decode_attention(q, dual(k), v, table, lens),
                 lambda: F.prompt_attention(q, k, dual(v), table, lens, off), lambda: F.kv_append(dual(x), k, v, table, lens, n_heads=4),
                 lambda: F.kv_append(x, k, dual(v), table, lens, n_heads=4), lambda: F.copy_pages(dual(k), _i32(0), _i32(1))]
        for call in calls:
            with pytest.raises(RuntimeError, match="no backward pass"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="no backward pass"):
                call()
        assert torch.equal(F.decode_attention(q, k, v, table, lens), want)
    with pytest.raises(RuntimeError, match="no backward pass"):
        torch.func.jvp(lambda t: F.decode_attention(t, k, v, table, lens), (q,), (q,))


def test_copy_pages_own_copy_is_a_source_too():
    page = lambda *v: torch.tensor(v, dtype=torch.float32).view(-1, 1, 1, 1).expand(-1, 1, 4, 4).contiguous()
    for src, dst, want in (((0, 0), (0, 1), (0, 0, 2)), ((1, 1, 1), (2, 1, 0), (1, 1, 1))):
        assert torch.equal(F.copy_pages(page(0, 1, 2), _i32(*src), _i32(*dst)), page(*want))
    for src, dst in (((0, 1), (1, 1)), ((1, 0), (1, 1))):
        with pytest.raises(IndexError):
            F.copy_pages(page(0, 1, 2), _i32(*src), _i32(*dst))


@pytest.mark.parametrize("shape", [(0, 4, 1, 16, 16), (3, 0, 4, 1, 16, 16), (2, 4, 0, 16, 16), (2, 4, 1, 16, 0)])
def test_copy_pages_of_nothing(shape):
    """No layers, or pages without elements: nothing to copy, and the pairs are looked at all the same."""
    st = torch.zeros(shape)
    assert F.copy_pages(st, _i32(0, 1), _i32(2, 3)) is st
    with pytest.raises(IndexError):
        F.copy_pages(st, _i32(0), _i32(4))


def test_what_has_kernels():
    from incin_b200 import _native as nat
    from incin_b200.ops.paged import check_kernels
    for dtype in (torch.bfloat16, torch.float16):
        for D in (64, 128):
            check_kernels("x", dtype, D, 128)
    for dtype, D, group in ((torch.float32, 64, 1), (torch.float64, 128, 1), (torch.bfloat16, 32, 1), (torch.float16, 256, 1), (torch.bfloat16, 64, 129)):
        with pytest.raises(nat.NativeError, match="x: "):
            check_kernels("x", dtype, D, group)
