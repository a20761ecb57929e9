"""CPU tests of the paged caches' host side: what the classes and the C entries refuse, ahead of any launch, what
traced and compiled programs hold, packed structures and layouts."""

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from gdl_amd import _native
from gdl_amd import functional as F

F32, BF16, F16, I8, E4 = torch.float32, torch.bfloat16, torch.float16, torch.int8, torch.float8_e4m3fn
T, B, H, HK, D = 20, 3, 4, 2, 16


def _cache(stored=F32, pages=6, page=64, d=D):
    cache = F.PagedCache.empty(pages, HK, d, page=page, dtype=stored, device="cpu")
    for t in (cache.k, cache.v, cache.k_scale, cache.v_scale):
        if t is not None:
            t.view(torch.uint8).zero_()
    return cache


# ------------------------------------------------------------------ the class ---


@pytest.mark.parametrize("stored,blk", [(F32, 16), (BF16, 32), (F16, 32), (I8, 64), (E4, 64)])
def test_layout(stored, blk):
    cache = _cache(stored, page=192)
    assert cache.k.shape == (6, HK, 192, D) and cache.v.shape == (6, HK, 192 // blk, D, blk)
    assert cache.page == 192 and cache.kv_heads == HK and cache.head_dim == D
    assert (cache.k_scale is None) == (stored not in (I8, E4)) and (stored not in (I8, E4) or cache.v_scale.shape == (6, HK, 192))


@pytest.mark.parametrize("kw", [dict(pages=0), dict(kv_heads=0), dict(page=0), dict(page=96), dict(page=32), dict(head_dim=12), dict(head_dim=136),
                                dict(head_dim=24, dtype=I8), dict(head_dim=0), dict(page=(1 << 20) + 64)])
def test_sizes_are_refused(kw):
    args = dict(pages=2, kv_heads=1, head_dim=16, page=64, dtype=F32, device="meta")
    with pytest.raises(ValueError):
        F.PagedCache.empty(**{**args, **kw})


def test_types_are_refused():
    with pytest.raises(TypeError):
        F.PagedCache.empty(2, 1, 16, dtype=torch.float64, device="cpu")
    with pytest.raises(TypeError):
        F.PagedCache(torch.zeros(2, 1, 64, 16), torch.zeros(2, 1, 2, 16, 32, dtype=F16))
    cache = _cache()
    x, table = torch.zeros(T, HK, D), torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(TypeError):
        cache.write(x.half(), x.half(), table)
    with pytest.raises(TypeError):
        cache.write(x, x, table.long())
    with pytest.raises(TypeError):
        cache.read(table, None, 5, dtype=BF16)
    with pytest.raises(TypeError):
        _cache(I8).read(table, None, 5, dtype=torch.float64)
    with pytest.raises(TypeError):
        F.paged_attention(x.bfloat16(), cache, table)
    with pytest.raises(TypeError):
        F.paged_attention_step(x[:1].bfloat16(), x[:1], x[:1], cache, table, torch.zeros(1, dtype=torch.int64))


def test_tensors_are_refused():
    k, v, s = torch.zeros(2, 1, 64, 16), torch.zeros(2, 1, 4, 16, 16), torch.zeros(2, 1, 64)
    F.PagedCache(k, v)
    for bad in ((k, v[:1]), (k, v.transpose(1, 2)), (k[0], v), (k.transpose(2, 3), v), (k, v, s, s.clone()),
                (torch.zeros(2, 1, 128, 16)[:, :, :64], v), (k, k.view(2, 1, 4, 16, 16)), (k.clone().requires_grad_(), v)):
        with pytest.raises(ValueError):
            F.PagedCache(*bad)
    whole = torch.zeros(4 * 1024 + 1)
    with pytest.raises(ValueError):  # not on 16 bytes
        F.PagedCache(whole[1:2049].view(2, 1, 64, 16), v)
    with pytest.raises(ValueError):  # half shared
        F.PagedCache(whole[:2048].view(2, 1, 64, 16), whole[1000:3048].view(2, 1, 4, 16, 16))
    k8, v8 = torch.zeros(2, 1, 64, 16, dtype=I8), torch.zeros(2, 1, 1, 16, 64, dtype=I8)
    F.PagedCache(k8, v8, s, s.clone())
    for bad in ((k8, v8), (k8, v8, s), (k8, v8, s, s), (k8, v8, s.half(), s.half().clone()), (k8, v8, s[:1], s)):
        with pytest.raises(ValueError):
            F.PagedCache(*bad)


def test_calls_are_refused():
    cache, x, table = _cache(), torch.zeros(T, HK, D), torch.zeros(B, 2, dtype=torch.int32)
    ptr, start, q = torch.tensor([0, 5, 5, T]), torch.zeros(B, dtype=torch.int64), torch.zeros(T, H, D)
    for args in ((x, x[:, :1], table, ptr), (x[..., :8], x[..., :8], table, ptr), (x, x, table), (x, x, table, ptr[:3]), (x, x, table[:, :0], ptr),
                 (x, x, table[0], ptr), (x, x, table, ptr.float()), (x, x, table, ptr, start[:2]), (x, x, table, ptr, start.float()),
                 (x, x, table, ptr.view(2, 2))):
        with pytest.raises(ValueError):
            cache.write(*args)
    for args in ((table, ptr, -1), (table, None, 4), (table[:2], ptr, 4)):
        with pytest.raises(ValueError):
            cache.read(*args)
    for args in ((q[:, :3], cache, table, ptr), (q[:, 0], cache, table, ptr), (q[..., :8], cache, table, ptr), (q, cache, table), (q, cache, table[:1], ptr),
                 (q[:, :0], cache, table, ptr)):
        with pytest.raises(ValueError):
            F.paged_attention(*args)
    for bias in (torch.zeros(8), torch.zeros(8, H + 1)):
        with pytest.raises(ValueError):
            F.paged_attention(q, cache, table, ptr, bias=bias)
    q, k, pos = q[:B], x[:B], start
    for args in ((q, k[:2], k[:2], table, pos), (q, k, k, table[:2], pos), (q, k, k, table, pos[:2]), (q, k, k, table, pos.float()),
                 (q[:, :3], k, k, table, pos), (q, k[:, :1], k[:, :1], table, pos)):
        with pytest.raises(ValueError):
            F.paged_attention_step(*args[:3], cache, *args[3:])


def test_gradients_are_refused():
    cache, table = _cache(), torch.zeros(1, 2, dtype=torch.int32)
    x, q = torch.zeros(1, HK, D), torch.zeros(1, H, D, requires_grad=True)
    for call in (lambda: cache.write(x.clone().requires_grad_(), x, table), lambda: F.paged_attention(q, cache, table),
                 lambda: F.paged_attention_step(q, x, x, cache, table, torch.zeros(1, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="no backward"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="GPU only"):
            call()


def test_cpu_tensors_are_refused():
    cache, table = _cache(E4), torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU only"):
        cache.read(table, None, 3)


# --------------------------------------------------------------- the C entries ---


def _pool(k=4096, v=1 << 20, k_scale=0, v_scale=0, table=4096, stride=2, pages=6, columns=2, stored=0, heads=HK, d=D, page=64):
    return _native.pack_paged(k, v, k_scale, v_scale, table, stride, pages, columns, stored, heads, d, page)


def _step(pool=None, q=4096, strides=(H * D, D) * 3, pos=4096, bias=0, lut=0, batch=2, dtype=0, heads=H, buckets=0, maxd=0):
    return _native.pack_paged_step(pool or _pool(), q, q, q, *strides, pos, bias, lut, batch, dtype, 0, heads, buckets, maxd, 0.25)


def _prompt(pool=None, q=4096, strides=(H * D, D), ptr=4096, bias=0, lut=0, tokens=8, batch=2, dtype=0, heads=H, buckets=0, maxd=0):
    return _native.pack_paged_prompt(pool or _pool(), q, *strides, ptr, 0, bias, lut, tokens, batch, dtype, 0, heads, buckets, maxd, 0.25)


def _refused(status, part):
    assert status != 0
    assert part in _native.lib().geo_last_error().decode(), _native.lib().geo_last_error()


def test_structures_fill_the_header_s():
    assert len(_pool()) == 80 and len(_step()) == 208 and len(_prompt()) == 176


BAD_POOLS = [(dict(stored=2), "type code 2"), (dict(stored=6), "type code 6"), (dict(heads=0), "key heads"), (dict(d=12), "head size 12"),
             (dict(d=136), "head size 136"), (dict(d=24, stored=4, k_scale=4096, v_scale=8192), "multiple of 16"), (dict(page=32), "pages of 32"),
             (dict(page=100), "pages of 100"), (dict(page=1 << 21), "pages of"), (dict(pages=0), "0 pages"), (dict(pages=1 << 31), "pages"),
             (dict(columns=0), "0 columns"), (dict(columns=1 << 24), "columns"), (dict(columns=(1 << 63) - 1), "columns"), (dict(k=0), "null pool"),
             (dict(v=8), "on 16 bytes"), (dict(v=4096), "one for both"), (dict(stored=4), "needs scales"),
             (dict(stored=5, k_scale=4096, v_scale=4096), "needs scales"), (dict(table=0), "null table")]


@pytest.mark.parametrize("change,part", BAD_POOLS)
def test_pools_are_refused(change, part):
    lib, pool = _native.lib(), _pool(**change)
    _refused(lib.geo_paged_write(pool, 0, 4096, 4096, 32, 16, 32, 16, 4096, None, 8, 2, None), part)
    _refused(lib.geo_paged_read(pool, 0, 4096, None, 8, 2, 4096, 8192, None), part)
    _refused(lib.geo_paged_attention_step(_step(pool), 4096, None, 0, None), part)
    _refused(lib.geo_paged_attention(_prompt(pool), 4096, None, 0, None), part)


@pytest.mark.parametrize("tokens,batch,ptr,part", [(-1, 2, 4096, "tokens"), ((1 << 31) - 64, 2, 4096, "tokens"), (8, -1, 4096, "sequences"),
                                                   (8, 1 << 30, 4096, "sequences"), (8, 2, None, "without ptr"), (8, 0, 4096, "no sequence"),
                                                   ((1 << 31) - 65, 1, 4096, "too many workgroups")])
def test_spans_are_refused(tokens, batch, ptr, part):
    lib = _native.lib()
    _refused(lib.geo_paged_write(_pool(), 0, 4096, 4096, 32, 16, 32, 16, ptr, None, tokens, batch, None), part)
    _refused(lib.geo_paged_read(_pool(), 0, ptr, None, tokens, batch, 4096, 8192, None), part)
    _refused(lib.geo_paged_attention(_prompt(ptr=ptr or 0, tokens=tokens, batch=batch), 4096, None, 0, None), part)


def test_rows_are_refused():
    lib = _native.lib()
    for k, strides in ((0, (32, 16)), (4100, (32, 16)), (4096, (33, 16)), (4096, (32, 17))):
        _refused(lib.geo_paged_write(_pool(), 0, k, 4096, *strides, 32, 16, 4096, None, 8, 2, None), "16 bytes")
        _refused(lib.geo_paged_attention_step(_step(q=k, strides=strides * 3), 4096, None, 0, None), "16 bytes")
        _refused(lib.geo_paged_attention(_prompt(q=k, strides=strides), 4096, None, 0, None), "16 bytes")
    _refused(lib.geo_paged_read(_pool(), 0, 4096, None, 8, 2, 4096, 4096, None), "one output")
    _refused(lib.geo_paged_write(_pool(), 1, 4096, 4096, 32, 16, 32, 16, 4096, None, 8, 2, None), "type code 1, a pool of 0")
    _refused(lib.geo_paged_write(_pool(stored=4, k_scale=4096, v_scale=8192), 4, 4096, 4096, 32, 16, 32, 16, 4096, None, 8, 2, None), "type code 4")


@pytest.mark.parametrize("change,part", [(dict(heads=5), "no multiple"), (dict(heads=1 << 20), "below 2^20"), (dict(batch=-1), "heads"),
                                         (dict(dtype=1), "type code 1"), (dict(pos=0), "null output or positions"),
                                         (dict(bias=4096, lut=4096, buckets=257, maxd=128), "257 buckets"),
                                         (dict(bias=4096, lut=4096, buckets=32, maxd=1025), "distance 1025"), (dict(bias=4096, buckets=8, maxd=9), "bias of")])
def test_steps_are_refused(change, part):
    _refused(_native.lib().geo_paged_attention_step(_step(**change), 4096, None, 0, None), part)


@pytest.mark.parametrize("change,part", [(dict(heads=5), "no multiple"), (dict(heads=1 << 20), "below 2^20"), (dict(dtype=1), "type code 1"),
                                         (dict(bias=4096, lut=4096, buckets=257, maxd=128), "257 buckets"),
                                         (dict(bias=4096, lut=4096, buckets=32, maxd=1025), "distance 1025")])
def test_prompts_are_refused(change, part):
    _refused(_native.lib().geo_paged_attention(_prompt(**change), 4096, None, 0, None), part)


def test_workspaces():
    lib = _native.lib()
    long = _pool(columns=4000, stride=4000)
    for args, size, call in ((_step(long), lib.geo_paged_attention_step_workspace_bytes, lib.geo_paged_attention_step),
                             (_prompt(long), lib.geo_paged_attention_workspace_bytes, lib.geo_paged_attention)):
        need = size(args)
        assert need > 0
        _refused(call(args, 4096, 4096, need - 1, None), "needed")
        _refused(call(args, 4096, None, need, None), "needed")
    assert lib.geo_paged_attention_step_workspace_bytes(_step()) == 0 and lib.geo_paged_attention_workspace_bytes(_prompt()) == 0
    for bad in (dict(columns=(1 << 63) - 1), dict(page=0), dict(page=-64), dict(heads=0), dict(heads=-1), dict(columns=-5)):
        pool = _pool(**bad)
        assert lib.geo_paged_attention_step_workspace_bytes(_step(pool)) == 0 and lib.geo_paged_attention_workspace_bytes(_prompt(pool)) == 0
    for bad in (dict(heads=0), dict(heads=-4), dict(batch=1 << 40), dict(heads=(1 << 31) - 2)):
        assert lib.geo_paged_attention_step_workspace_bytes(_step(long, **bad)) == 0
        assert lib.geo_paged_attention_workspace_bytes(_prompt(long, **bad)) == 0


def test_nothing_to_do_is_done():
    lib = _native.lib()
    assert lib.geo_paged_write(_pool(), 0, None, None, 0, 0, 0, 0, 4096, None, 0, 2, None) == 0
    assert lib.geo_paged_read(_pool(), 0, 4096, None, 0, 2, None, None, None) == 0
    assert lib.geo_paged_attention_step(_step(q=0, batch=0), None, None, 0, None) == 0
    assert lib.geo_paged_attention(_prompt(q=0, tokens=0), None, None, 0, None) == 0


# ------------------------------------------------------ programs without pointers ---


def _write(k, v, kc, vc, ks, vs, table, ptr, start):
    F.PagedCache(kc, vc, ks, vs).write(k, v, table, ptr, start)
    return kc.float() + vc.view(kc.shape).float()


def _read(kc, vc, ks, vs, table, ptr):
    return F.PagedCache(kc, vc, ks, vs).read(table, ptr, T, dtype=F32)


def _attend(q, kc, vc, ks, vs, table, ptr, start, bias):
    return F.paged_attention(q, F.PagedCache(kc, vc, ks, vs), table, ptr, start, bias=bias, max_distance=9)


def _attend_step(q, k, v, kc, vc, ks, vs, table, pos, bias):
    return F.paged_attention_step(q, k, v, F.PagedCache(kc, vc, ks, vs), table, pos, bias=bias, max_distance=9)


def _pools():
    cache = _cache(I8)
    cache.k.random_(-127, 128), cache.v.random_(-127, 128), cache.k_scale.uniform_(), cache.v_scale.uniform_()
    return cache.k, cache.v, cache.k_scale, cache.v_scale


def _rows(n=T):
    return [torch.randn(n, HK, D) for _ in range(2)]


def _table():
    return torch.arange(2 * B, dtype=torch.int32).view(B, 2)


PTR, START = torch.tensor([0, 10, 10, T]), torch.tensor([3, 0, 60])
CALLS = {"paged_write": (_write, lambda: (*_rows(), *_pools(), _table(), PTR, START)),
         "paged_read": (_read, lambda: (*_pools(), _table(), PTR)),
         "paged_attention": (_attend, lambda: (torch.randn(T, H, D), *_pools(), _table(), PTR, START, torch.randn(8, H))),
         "paged_attention_step": (_attend_step, lambda: (torch.randn(B, H, D), *_rows(B), *_pools(), _table(), torch.tensor([70, 0, 127]), torch.randn(8, H)))}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("mode", ["fake", "symbolic"])
def test_a_trace_holds_the_op(name, mode):
    call, args = CALLS[name]
    assert f"geoembodied.{name}." in make_fx(call, tracing_mode=mode)(*args()).code


@pytest.mark.parametrize("name", CALLS)
def test_compilation_takes_the_call_whole(name):
    call, args = CALLS[name]
    seen = []

    def backend(module, inputs):
        seen.append(module.print_readable(print_output=False))
        raise RuntimeError("the backend stops before anything runs")

    torch._dynamo.reset()
    with pytest.raises(Exception):
        torch.compile(call, backend=backend, fullgraph=True)(*args())
    assert len(seen) == 1 and name in seen[0]


@pytest.mark.parametrize("name", [n for n in CALLS if n != "paged_read"])
def test_forward_mode_is_refused(name):
    call, args = CALLS[name]
    inputs = list(args())
    with torch.autograd.forward_ad.dual_level():
        inputs[0] = torch.autograd.forward_ad.make_dual(inputs[0], torch.ones_like(inputs[0]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(*inputs)


def test_bucket_configurations_are_checked_when_traced():
    args = CALLS["paged_attention"][1]()
    with pytest.raises(ValueError):
        make_fx(lambda q, kc, vc, ks, vs, table, ptr, start, bias: F.paged_attention(q, F.PagedCache(kc, vc, ks, vs), table, ptr, start, bias=bias,
                                                                                     max_distance=2000), tracing_mode="fake")(*args)


def test_module_paths():
    import geoembodied  # noqa: F401
    from geoembodied.functional.paged import PagedCache, paged_attention, paged_attention_step

    assert PagedCache is F.PagedCache and paged_attention is F.paged_attention and paged_attention_step is F.paged_attention_step
