"""The paged cache's operators on the host: struct layouts of the binding, and refusals, which come before any device work."""
import ctypes as C
import os
import subprocess

import pytest
import torch

import tsn
from tsn import paged_ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {"tsn_paged": tsn.Paged, "tsn_cache_append_args": tsn.CacheAppendArgs, "tsn_paged_attn_args": tsn.PagedAttnArgs,
           "tsn_sparse_attn_args": tsn.SparseAttnArgs}


def test_binding_has_the_headers_layouts(tmp_path):
    lines = []
    for name, cls in STRUCTS.items():
        lines.append(f'printf("{name} %zu", sizeof({name}));')
        lines += [f'printf(" %zu", offsetof({name}, {f[0]}));' for f in cls._fields_]
        lines.append('printf("\\n");')
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "tsn.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0;\n}\n")
    exe = str(tmp_path / "layout")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    for line in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.splitlines():
        name, *numbers = line.split()
        cls = STRUCTS[name]
        assert [int(n) for n in numbers] == [C.sizeof(cls)] + [getattr(cls, f[0]).offset for f in cls._fields_], name


A = 1 << 20   # an aligned address that nothing reads


def cache(**change):
    c = dict(B=2, N=5, P=8, M=4, page=16, Hk=2, D=64, type=1, k=tsn.Heads(A, 2048, 128, 64), v=tsn.Heads(A, 2048, 128, 64), table=A, table_sb=4,
             len=A, q_start=A)
    c.update(change)
    return tsn.Paged(**c)


def rows(H=4, **change):
    r = dict(p=A, sb=H * 64, st=64)
    r.update(change)
    return tsn.Rows(**r)


def refused(name, args, plan=None):
    """The refusal of a call without a device, or None where its arguments are fine."""
    fn = getattr(tsn.lib(), name)
    rc = fn(None, plan, C.byref(args)) if name == "tsn_cache_append" else fn(None, C.byref(args))
    assert rc == 1
    why = tsn.lib().tsn_last_error().decode()
    return None if why == "null argument" else why


CACHE = [dict(type=0), dict(type=3), dict(page=0), dict(page=8), dict(page=48), dict(page=2048), dict(Hk=0), dict(Hk=70000), dict(B=70000),
         dict(N=2 ** 30 + 1), dict(P=2 ** 31), dict(M=2 ** 26 + 1), dict(M=2 ** 31), dict(q_start=None), dict(len=None), dict(table=None),
         dict(k=tsn.Heads(None, 2048, 128, 64)), dict(v=tsn.Heads(A + 2, 2048, 128, 64)), dict(k=tsn.Heads(A, 2044, 128, 64)),
         dict(k=tsn.Heads(A, 2048, 0, 64)), dict(v=tsn.Heads(A, 2048, 128, -64)), dict(v=tsn.Heads(A, 2 ** 40, 128, 64)), dict(len=A + 2),
         dict(table_sb=-4)]


@pytest.mark.parametrize("change", CACHE, ids=[str(sorted(c)) + str(i) for i, c in enumerate(CACHE)])
def test_caches(change):
    assert refused("tsn_paged_attn", tsn.PagedAttnArgs(c=cache(**change), H=4, causal=1, q=rows(), out=rows()))
    assert refused("tsn_sparse_attn", tsn.SparseAttnArgs(c=cache(**change), H=4, picks=4, first=1, last=1, q=rows(), out=rows(), means=rows(2), chosen=A))
    assert refused("tsn_cache_append", append(c=cache(**change)), plan())


def plan(D=64, pairs=(32,), layout=0):
    p, n = tsn.RopePlan(), len(pairs)
    tsn.check(tsn.lib().tsn_rope_plan(D, n, (C.c_uint32 * n)(*pairs), (C.c_double * n)(*[1e4] * n), (C.c_double * n)(*[1.0] * n), layout, C.byref(p)))
    return p


def append(**change):
    a = dict(c=cache(), Hq=4, xtype=1, eps=1e-6, q=rows(), k=rows(2), v=rows(2), q_out=rows(), means=rows(2))
    a.update(change)
    return tsn.CacheAppendArgs(**a)


APPEND = [dict(xtype=2), dict(xtype=5), dict(eps=-1.0), dict(eps=float("nan")), dict(Hq=70000), dict(q_out=rows(p=None)), dict(k=rows(p=None)),
          dict(v=rows(p=None)), dict(q=rows(p=A + 8)), dict(k=rows(sb=130)), dict(v=rows(st=68)), dict(q_out=rows(sb=0)), dict(means=rows(p=A + 4)),
          dict(means=rows(sb=0)), dict(xtype=0, q=rows(sb=254)), dict(pos=A + 1), dict(q_norm=A + 2), dict(c=cache(D=128))]


@pytest.mark.parametrize("change", APPEND, ids=[str(sorted(c)) + str(i) for i, c in enumerate(APPEND)])
def test_appending(change):
    assert refused("tsn_cache_append", append(**change), plan())


def test_plans():
    assert refused("tsn_cache_append", append(), plan()) is None
    assert refused("tsn_cache_append", append(), plan(pairs=(8, 8)))          # positions are wanted
    assert refused("tsn_cache_append", append(pos=A), plan(pairs=(8, 8))) is None
    assert refused("tsn_cache_append", append(c=cache(D=60)), plan(D=60, pairs=(8,)))
    for change in (dict(P=2 ** 31), dict(P=33), dict(D=0), dict(D=258), dict(axes=0), dict(axes=5), dict(layout=2)):
        p = plan()
        for name, value in change.items():
            setattr(p, name, value)
        assert refused("tsn_cache_append", append(), p)
    p = plan()
    p.axis[3] = 1
    assert refused("tsn_cache_append", append(), p)


def test_attention():
    attn = lambda **x: refused("tsn_paged_attn", tsn.PagedAttnArgs(**{**dict(c=cache(), H=4, causal=1, q=rows(), out=rows()), **x}))  # noqa: E731
    sparse = lambda **x: refused("tsn_sparse_attn", tsn.SparseAttnArgs(  # noqa: E731
        **{**dict(c=cache(), H=4, picks=4, first=1, last=1, q=rows(), out=rows(), means=rows(2), chosen=A), **x}))
    assert attn() is None and sparse() is None
    for f in (attn, sparse):
        for change in (dict(H=0), dict(H=5), dict(H=258), dict(H=2 ** 31), dict(c=cache(D=96)), dict(c=cache(D=256)), dict(scale=-1.0),
                       dict(scale=float("nan")), dict(scale=float("inf")), dict(q=rows(p=None)), dict(out=rows(p=None)), dict(out=rows(sb=0)),
                       dict(out=rows(st=0)), dict(q=rows(sb=252)), dict(out=rows(p=A + 8)), dict(c=cache(N=2 ** 30), H=16)):
            assert f(**change), change
        assert f(q=rows(sb=0)) is None   # one query for all
        assert f(c=cache(N=0)) is None and f(c=cache(N=0, B=0)) is None and f(c=cache(P=0)) is None and f(c=cache(M=0, table=None)) is None
    assert attn(causal=0, window=3) and attn(window=2 ** 30 + 1) and attn(causal=0) is None and attn(window=2 ** 30, most=2 ** 31) is None
    for change in (dict(picks=0), dict(picks=1), dict(picks=1025), dict(last=0), dict(first=4), dict(first=2 ** 32 - 1, last=2), dict(c=cache(M=16385)),
                   dict(means=rows(p=None)), dict(chosen=None), dict(chosen=A + 2)):
        assert sparse(**change), change


class Host:
    """A handle whose tensors lie in host memory."""
    ordinal = -1
    h = C.c_void_p(0)


def tensors(N=5, H=4, D=64, B=2, dtype=torch.float16):
    z = lambda *s, t=dtype: torch.zeros(s, dtype=t)  # noqa: E731
    i = lambda *s: z(*s, t=torch.int32)  # noqa: E731
    return dict(q=z(N, H, D), k_pages=z(8, 16, 2, D), v_pages=z(8, 16, 2, D), table=i(B, 4), lens=i(B), out=z(N, H, D), q_start=i(B + 1))


def bad_batches():
    z, i = torch.zeros, torch.int32
    yield dict(k_pages=z(8, 16, 2, 32).half())
    yield dict(k_pages=z(8, 16, 2, 64))
    yield dict(v_pages=z(8, 16, 3, 64).half())
    yield dict(v_pages=z(8, 16, 2, 64).bfloat16())
    yield dict(k_pages=z(8, 16, 64, 2).half().transpose(2, 3))
    yield dict(table=z(2, 4))
    yield dict(table=z(4, 2, dtype=i).t())
    yield dict(table=z(3, 4, dtype=i))
    yield dict(lens=z(3, dtype=i))
    yield dict(lens=z(2, dtype=torch.int64))
    yield dict(lens=z(4, dtype=i)[::2])
    yield dict(q_start=z(2, dtype=i))
    yield dict(q_start=None)
    yield dict(q=z(5, 4, 64).bfloat16())
    yield dict(q=z(5, 4, 32).half())
    yield dict(q=z(20, 64).half())
    yield dict(out=z(4, 4, 64).half())
    yield dict(out=z(5, 4, 64))
    yield dict(out=z(5, 64, 4).half().transpose(1, 2))
    yield dict(out=torch.empty(5, 4, 64, dtype=torch.float16, device="meta"))


@pytest.mark.parametrize("change", list(bad_batches()), ids=lambda c: next(iter(c)))
def test_tensors_that_do_not_fit(change):
    op = tsn.PagedAttention(Host, 64)
    op._call = lambda dev, args: 0
    op(**tensors())
    with pytest.raises((ValueError, TypeError)):
        op(**{**tensors(), **change})
    op(**tensors())   # and the refused call left no form behind
    if "out" not in change:
        t = {**tensors(), **change}
        sparse = tsn.SparseAttention(Host, 64, 3)
        sparse._call = lambda dev, args: 0
        with pytest.raises((ValueError, TypeError)):
            sparse(means=torch.zeros(8, 2, 64).half(), chosen=torch.zeros(5, 2, 3, dtype=torch.int32), **t)


def test_every_operator_sets_its_addresses():
    at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    op = paged_ops.PagedAttention(Host, 64)
    op._call = lambda dev, args: 0
    checks, check = [], op._check
    op._check = lambda *t: (checks.append(1), check(*t))
    for _ in range(3):
        t = tensors()
        op(**t, window=3, most=7)
        a = op._a
        assert [a.q.p, a.out.p, a.c.k.p, a.c.v.p, a.c.table, a.c.len, a.c.q_start] == \
            [at(t[n]) for n in ("q", "out", "k_pages", "v_pages", "table", "lens", "q_start")]
        assert (a.c.B, a.c.N, a.c.P, a.c.M, a.c.page, a.c.Hk, a.c.D, a.c.type, a.H, a.causal, a.window, a.most) == (2, 5, 8, 4, 16, 2, 64, 1, 4, 1, 3, 7)
    assert len(checks) == 1
    t = tensors(N=2)
    t["q_start"] = None
    op(**t)
    assert op._a.c.q_start is None and op._a.c.N == 2
    sparse = paged_ops.SparseAttention(Host, 64, 3, first=0)
    sparse._call = lambda dev, args: 0
    append = paged_ops.CacheAppend(Host, 64, (32,))
    append._call = lambda dev, plan, args: 0
    for _ in range(2):
        t = tensors()
        means, chosen = torch.zeros(8, 2, 64).half(), torch.zeros(5, 2, 3, dtype=torch.int32)
        sparse(means=means, chosen=chosen, **t)
        a = sparse._a
        assert [a.q.p, a.out.p, a.means.p, a.chosen, a.c.k.p, a.c.v.p, a.c.table, a.c.len, a.c.q_start] == \
            [at(x) for x in (t["q"], t["out"], means, chosen, t["k_pages"], t["v_pages"], t["table"], t["lens"], t["q_start"])]
        k, v, pos, q_out = torch.zeros(5, 2, 64), torch.zeros(5, 2, 64), torch.zeros(5, 1, dtype=torch.int32), t.pop("out")
        q = t.pop("q").float()
        append(q, k, v, q_out=q_out, pos=pos, means=means, **t)
        a = append._a
        assert [a.q.p, a.k.p, a.v.p, a.q_out.p, a.pos, a.means.p, a.c.k.p, a.c.v.p, a.c.table, a.c.len, a.c.q_start] == \
            [at(x) for x in (q, k, v, q_out, pos, means, t["k_pages"], t["v_pages"], t["table"], t["lens"], t["q_start"])]
        assert (a.Hq, a.xtype, a.c.type) == (4, 0, 1)
    append(None, k, v, **t)
    assert [append._a.q.p, append._a.q_out.p, append._a.pos, append._a.means.p, append._a.Hq] == [None, None, None, None, 0]


def test_appended_tensors_that_do_not_fit():
    op = tsn.CacheAppend(Host, 64, (8, 8))
    op._call = lambda dev, plan, args: 0
    t = tensors()
    base = dict(q=t["q"], k=torch.zeros(5, 2, 64).half(), v=torch.zeros(5, 2, 64).half(), q_out=t["out"], pos=torch.zeros(5, 2, dtype=torch.int32),
                **{n: t[n] for n in ("k_pages", "v_pages", "table", "lens", "q_start")})
    op(**base)
    z = torch.zeros
    for change in (dict(pos=None), dict(pos=z(5, 1, dtype=torch.int32)), dict(pos=z(5, 2)), dict(k=z(5, 3, 64).half()), dict(k=z(5, 2, 64)),
                   dict(v=z(5, 2, 64)), dict(q=z(4, 4, 64).half()), dict(q=z(5, 4, 64)), dict(q_out=z(5, 3, 64).half()), dict(q_out=z(5, 4, 64)),
                   dict(means=z(8, 2, 64)), dict(means=z(7, 2, 64).half()), dict(k=z(5, 2, 64).bfloat16(), v=z(5, 2, 64).bfloat16())):
        with pytest.raises((ValueError, TypeError)):
            op(**{**base, **change})
    with pytest.raises(TypeError):   # in place only where the types agree
        op(**{**base, "q": z(5, 4, 64), "k": z(5, 2, 64), "v": z(5, 2, 64), "q_out": None})
    with pytest.raises(ValueError):
        tsn.CacheAppend(Host, 64, (8,), layout="other")
    with pytest.raises(tsn.TsnError):
        tsn.CacheAppend(Host, 64, (33,))
