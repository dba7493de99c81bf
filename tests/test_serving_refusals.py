"""What the serving calls refuse, and host-side checks of their C entries (no
GPU needed)."""
import ctypes as C

import pytest
import torch

import b200decode
from b200decode import _lib


def cross_args(**kw):
    a = _lib.CrossArgs()
    a.num_tokens, a.num_groups, a.query_len = 12, 4, 3
    a.num_q_heads, a.num_kv_heads, a.head_dim = 32, 8, 128
    a.page_size, a.max_pages_per_seq = 16, 64
    a.q_dtype = a.kv_dtype = _lib.B2D_BF16
    a.num_ctas = 148
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(head_dim=96), -2), (dict(head_dim=0), -2), (dict(num_q_heads=30), -1), (dict(num_kv_heads=0), -1),
    (dict(num_q_heads=8 * 33), -2), (dict(q_dtype=_lib.B2D_FP8_E4M3), -2), (dict(kv_dtype=_lib.B2D_FP16), -2),
    (dict(page_size=0), -1), (dict(max_pages_per_seq=0), -1), (dict(num_tokens=-1), -1), (dict(num_groups=-1), -1),
    (dict(query_len=-1), -1), (dict(kv_layout=9), -1), (dict(wait_limit_us=-1), -1), (dict(flags=1), -1),
    (dict(kv_layout=_lib.B2D_KV_VLLM, kv_dtype=_lib.B2D_FP8_E4M3), -2),
    (dict(kv_layout=_lib.B2D_KV_VLLM, page_size=8), -2),
    (dict(max_pages_per_seq=1 << 28), -8), (dict(page_size=1 << 25), -8),
    (dict(num_tokens=1 << 30, max_pages_per_seq=1 << 20), -8),   # the chunk line would pass 32 bits
])
def test_cross_sizes_refused(kw, code):
    lib, n = _lib.load(), C.c_size_t(0)
    assert lib.b2d_cross_workspace_bytes(C.byref(cross_args(**kw)), C.byref(n)) == code
    assert lib.b2d_cross_attention(C.byref(cross_args(**kw)), None) == code


def test_cross_pointers_and_strides_refused():
    lib, n = _lib.load(), C.c_size_t(0)
    assert lib.b2d_cross_workspace_bytes(C.byref(cross_args()), C.byref(n)) == 0
    assert n.value > _lib.B2D_WORKSPACE_HEADER_BYTES
    assert lib.b2d_cross_workspace_bytes(None, C.byref(n)) == -1
    assert lib.b2d_cross_workspace_bytes(C.byref(cross_args()), None) == -1
    assert lib.b2d_cross_attention(None, None) == -1
    assert lib.b2d_cross_attention(C.byref(cross_args()), None) == -1                  # null pointers
    assert lib.b2d_cross_attention(C.byref(cross_args(num_tokens=0)), None) == 0       # nothing to do
    assert lib.b2d_cross_attention(C.byref(cross_args(num_groups=0)), None) == 0
    good = dict(q=256, k_cache=256, v_cache=256, kv_lens=256, block_table=256, out=256, num_pages=9,
                q_stride_t=4096, q_stride_h=128, out_stride_t=4096, out_stride_h=128,
                k_stride_page=16384, k_stride_tok=1024, k_stride_head=128,
                v_stride_page=16384, v_stride_tok=1024, v_stride_head=128)
    call = lambda **kw: lib.b2d_cross_attention(C.byref(cross_args(**{**good, **kw})), None)  # noqa: E731
    assert call() == -4                                     # no workspace
    assert call(workspace=256, workspace_bytes=n.value - 1) == -4
    assert call(workspace=264, workspace_bytes=n.value) == -3
    assert call(q=264) == -3 and call(k_cache=257) == -3 and call(out=258) == -3
    assert call(q_stride_t=4097) == -3 and call(k_stride_tok=1028) == -3 and call(v_stride_page=0) == -3
    assert call(num_pages=0) == -1 and call(query_len=4) == -1


def shared_args(**kw):
    a = _lib.SharedPrefixArgs()
    o = a.own
    o.batch, o.num_q_heads, o.num_kv_heads, o.head_dim = 8, 32, 8, 128
    o.page_size, o.max_pages_per_seq = 16, 64
    o.q_dtype = o.kv_dtype = _lib.B2D_BF16
    o.num_ctas = 148
    a.num_groups, a.prefix_max_pages = 1, 100
    for k, v in kw.items():
        setattr(o if hasattr(o, k) else a, k, v)
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(head_dim=96), -2), (dict(batch=-1), -1), (dict(num_groups=-1), -1), (dict(prefix_max_pages=0), -1),
    (dict(num_groups=4097), -8), (dict(prefix_max_pages=1 << 28), -8), (dict(max_pages_per_seq=0), -1),
    (dict(kv_dtype=_lib.B2D_FP16), -2), (dict(head_dim=192, kv_dtype=_lib.B2D_FP8_E4M3), -2),
])
def test_shared_sizes_refused(kw, code):
    lib, n = _lib.load(), C.c_size_t(0)
    assert lib.b2d_shared_prefix_workspace_bytes(C.byref(shared_args(**kw)), C.byref(n)) == code


def test_shared_calls_refused():
    lib, n = _lib.load(), C.c_size_t(0)
    assert lib.b2d_shared_prefix_workspace_bytes(C.byref(shared_args()), C.byref(n)) == 0
    # the own tokens' part: one fp32 copy of out at least
    assert n.value > 8 * 32 * 128 * 4
    call = lambda **kw: lib.b2d_decode_shared_prefix(C.byref(shared_args(**kw)), None)  # noqa: E731
    assert lib.b2d_decode_shared_prefix(None, None) == -1
    assert call() == -1 and call(batch=0) == 0
    assert call(flags=_lib.B2D_FLAG_SKIP_COMBINE) == -1 and call(num_groups=2) == -1


@pytest.mark.parametrize("kw,code", [
    (dict(num_states=0), -1), (dict(num_tokens=-1), -1), (dict(head_dim=12), -2), (dict(head_dim=1032), -2),
    (dict(in_dtype=_lib.B2D_FP8_E4M3), -2), (dict(out_dtype=_lib.B2D_FP16), -2), (dict(outs=None), -1),
    (dict(outs=264), -3), (dict(outs_stride_h=4), -3), (dict(out_stride_t=9), -3), (dict(num_tokens=0), 0),
])
def test_merge_refused(kw, code):
    a = _lib.MergeArgs()
    a.outs = a.lses = a.out = 256
    a.num_states, a.num_tokens, a.num_heads, a.head_dim = 2, 3, 4, 64
    for k, v in kw.items():
        setattr(a, k, v)
    assert _lib.load().b2d_merge_states(C.byref(a), None) == code


def test_pages_refused():
    lib = _lib.load()
    good = dict(cache_seqlens=256, block_table=256, block_table_stride=8, free_pages=256, free_count=256,
                seqlens_out=256, free_count_out=256, num_requests=4, max_pages_per_seq=8, page_size=16,
                free_capacity=10, workspace=256, workspace_bytes=_lib.B2D_WORKSPACE_HEADER_BYTES)
    for cls, fn, more in ((_lib.PlanAppendArgs, lib.b2d_plan_append, dict(slot_mapping=256, query_starts=256, max_tokens=4)),
                          (_lib.ReleaseArgs, lib.b2d_release_pages, dict(finished=256))):
        def call(**kw):
            a = cls()
            for k, v in {**good, **more, **kw}.items():
                setattr(a, k, v)
            return fn(C.byref(a), None)
        assert fn(None, None) == -1
        for k in ("num_requests", "free_capacity"):
            assert call(**{k: -1}) == -1
        for k in ("max_pages_per_seq", "page_size"):
            assert call(**{k: 0}) == -1
        for k in ("cache_seqlens", "block_table", "free_pages", "free_count", "seqlens_out", "free_count_out",
                  *(x for x in more if x != "max_tokens")):
            assert call(**{k: None}) == -1, k
        if fn is lib.b2d_plan_append:
            assert call(max_tokens=(1 << 30) + 1) == -8
        assert call(num_requests=16385) == -8 and call(max_pages_per_seq=1 << 28) == -8
        assert call(workspace=None) == -4 and call(workspace_bytes=100) == -4 and call(workspace=8) == -3


def test_cpu_tensors_refused():
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    kc = torch.zeros(1, 16, 1, 64, dtype=torch.bfloat16)
    one, bt = torch.ones(2, dtype=torch.int32), torch.zeros(2, 1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        b200decode.cross_attention(q, kc, kc, one, bt)
    with pytest.raises(RuntimeError, match="CUDA"):
        b200decode.decode_shared_prefix(q, kc, kc, one[:1], bt[:1], one, bt)
    with pytest.raises(RuntimeError, match="CUDA"):
        b200decode.merge_states(q[None].float(), torch.zeros(1, 2, 4))
    with pytest.raises(RuntimeError, match="CUDA"):
        b200decode.plan_append(one, bt, one, one[:1], 16)
    with pytest.raises(RuntimeError, match="CUDA"):
        b200decode.release_pages(one, bt, one.bool(), one, one[:1], 16)


class TestOnGpu:
    """Refusals of the Python layer that look at CUDA tensors; nothing is launched."""
    pytestmark = pytest.mark.gpu

    def args(self, cuda):
        bf = torch.bfloat16
        q = torch.zeros(5, 4, 64, dtype=bf, device=cuda)
        kc = torch.zeros(3, 16, 2, 64, dtype=bf, device=cuda)
        kl = torch.ones(2, dtype=torch.int32, device=cuda)
        bt = torch.zeros(2, 3, dtype=torch.int32, device=cuda)
        st = torch.tensor([0, 2, 5], dtype=torch.int32, device=cuda)
        return q, kc, kl, bt, st

    @pytest.mark.parametrize("change", [
        dict(q="float"), dict(kc="half"), dict(kl="long"), dict(bt="long"), dict(st="long"), dict(kl="short"),
        dict(st="short"), dict(bt="cpu"), dict(kc="cpu"), dict(q="2d"), dict(out="float"), dict(lse="half"),
        dict(kv_layout="XYZ"), dict(kc="narrow"), dict(q="heads")])
    def test_cross(self, cuda, change):
        q, kc, kl, bt, st = self.args(cuda)
        kw = {}
        (name, how), = change.items()
        if name == "out":
            kw["out"] = q.float()
        elif name == "lse":
            kw["lse"] = torch.zeros(5, 4, dtype=torch.half, device=cuda)
        elif name == "kv_layout":
            kw["kv_layout"] = how
        else:
            x = dict(q=q, kc=kc, kl=kl, bt=bt, st=st)
            t = x[name]
            x[name] = {"float": lambda: t.float(), "half": lambda: t.half(), "long": lambda: t.long(),
                       "short": lambda: t[:-1], "cpu": lambda: t.cpu(), "2d": lambda: t[0],
                       "narrow": lambda: t[..., :32], "heads": lambda: t[:, :3]}[how]()
            q, kc, kl, bt, st = (x[n] for n in ("q", "kc", "kl", "bt", "st"))
        with pytest.raises(ValueError):
            b200decode.cross_attention(q, kc, kc, kl, bt, query_starts=st, **kw)
        q, kc, kl, bt, st = self.args(cuda)
        with pytest.raises(ValueError, match="out must not be q"):
            b200decode.cross_attention(q, kc, kc, kl, bt, query_starts=st, out=q)

    def test_shared(self, cuda):
        q, kc, kl, bt, st = self.args(cuda)
        call = b200decode.decode_shared_prefix
        q = q[:2]
        with pytest.raises(ValueError, match="group_starts"):
            call(q, kc, kc, kl, bt, kl, bt)
        with pytest.raises(ValueError):
            call(q, kc, kc, kl, bt, kl, bt, group_starts=st[:2])
        with pytest.raises(ValueError):
            call(q, kc, kc, kl[:1], bt, kl, bt)
        with pytest.raises(ValueError):
            call(q, kc, kc, kl[:1].long(), bt[:1], kl, bt)
        with pytest.raises(ValueError):
            call(q, kc, kc, kl[:1], bt[:1].cpu(), kl, bt)
        with pytest.raises(ValueError):
            call(q, kc, kc, kl[:1], bt[:1], kl, bt, out=q.float())
        with pytest.raises(ValueError, match="out must not be q"):
            call(q, kc, kc, kl[:1], bt[:1], kl, bt, out=q)
        with pytest.raises(ValueError, match="one query token"):
            call(q[None], kc, kc, kl[:1], bt[:1], kl[:1], bt[:1])

    def test_merge(self, cuda):
        o, l = torch.zeros(2, 3, 4, 64, device=cuda), torch.zeros(2, 3, 4, device=cuda)
        call = b200decode.merge_states
        for bad in (lambda: call(o.double(), l), lambda: call(o, l.double()), lambda: call(o, l[:1]),
                    lambda: call(o[0], l[0]), lambda: call(o.half(), l, out=o[0].bfloat16()),
                    lambda: call(o, l, out=o[0]), lambda: call(o, l, lse=l[1]), lambda: call(o, l.cpu()),
                    lambda: call(o.transpose(2, 3), l)):
            with pytest.raises(ValueError):
                bad()

    def test_pages(self, cuda):
        i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=cuda)  # noqa: E731
        sl, bt, free, cnt = i32(4), i32(4, 6), i32(20), i32(1)
        call = b200decode.plan_append
        for bad in (lambda: call(sl.long(), bt, free, cnt, 16), lambda: call(sl, bt[:3], free, cnt, 16),
                    lambda: call(sl, bt, free.long(), cnt, 16), lambda: call(sl, bt, free, i32(2), 16),
                    lambda: call(sl, bt, free, cnt, 0), lambda: call(sl, bt, free, cnt, 16, new_tokens=sl),
                    lambda: call(sl, bt, free.cpu(), cnt, 16), lambda: call(sl, bt[:, ::2], free, cnt, 16),
                    lambda: call(sl, bt[:1].expand(4, 6), free, cnt, 16),
                    lambda: call(sl, bt, free, cnt, 16, slot_mapping=i32(4)),
                    lambda: call(sl, bt, free, cnt, 16, seqlens_out=i32(3))):
            with pytest.raises(ValueError):
                bad()
        for bad in (lambda: b200decode.release_pages(sl, bt, sl, free, cnt, 16),
                    lambda: b200decode.release_pages(sl, bt, sl[:3].bool(), free, cnt, 16)):
            with pytest.raises(ValueError):
                bad()
