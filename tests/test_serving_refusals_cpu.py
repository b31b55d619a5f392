"""CPU: what the serving operators refuse, before anything touches a device."""
import ctypes as C

import pytest
import torch

import flashmhf_b200 as fm
from flashmhf_b200 import _lib


def _pages(n=4, kv=2, P=16, hd=64):
    return fm.KVPages.empty(n, kv, P, hd, device="cpu")


def _x(*s):
    return torch.zeros(*s, dtype=torch.bfloat16)


def _i(*v):
    return torch.tensor(v, dtype=torch.int32)


def _append(**w):
    a = dict(pages=_pages(), k=_x(3, 2, 64), v=_x(3, 2, 64), cos=torch.ones(8, 32), sin=torch.ones(8, 32), lengths=_i(0, 1, 2),
             page_table=torch.zeros(3, 2, dtype=torch.int32))
    a.update(w)
    return fm.paged_append(**a)


def _attend(**w):
    a = dict(q=_x(3, 4, 64), pages=_pages(), lengths=_i(0, 1, 2), page_table=torch.zeros(3, 2, dtype=torch.int32))
    a.update(w)
    return fm.paged_attention(**a)


def _prompt(**w):
    a = dict(q=_x(5, 4, 64), k=_x(5, 2, 64), v=_x(5, 2, 64), cu_seqlens=_i(0, 2, 5))
    a.update(w)
    return fm.prompt_attention(**a)


BAD_POOLS = [(ValueError, _pages(hd=80)), (ValueError, _pages(P=24)), (ValueError, _pages()._replace(v=_pages(n=5).v)),
             (ValueError, _pages()._replace(k_scale=torch.ones(4, 3))), (TypeError, _pages()._replace(k_scale=torch.ones(4, 2).double())),
             (TypeError, _pages()._replace(k=_pages().k.view(torch.uint8))), (ValueError, _pages()._replace(k=_pages(P=128, hd=64).k[:, :, :16])),
             (ValueError, _pages()._replace(k=_pages(n=8).k[::2]))]


@pytest.mark.parametrize("error,more", [
    (ValueError, dict()),                                             # CPU tensors: there is no CPU path
    (ValueError, dict(k=_x(3, 3, 64))), (ValueError, dict(v=_x(2, 2, 64))), (ValueError, dict(k=_x(3, 2, 96))), (ValueError, dict(k=_x(3, 128))),
    (TypeError, dict(k=_x(3, 2, 64).float())), (TypeError, dict(q=_x(3, 2, 64).half())), (ValueError, dict(q=_x(4, 2, 64))),
    (ValueError, dict(q=_x(3, 0, 64))), (ValueError, dict(lengths=_i(0, 1))), (TypeError, dict(lengths=torch.zeros(3, dtype=torch.int64))),
    (ValueError, dict(page_table=torch.zeros(2, 2, dtype=torch.int32))), (TypeError, dict(page_table=torch.zeros(3, 2, dtype=torch.int64))),
    (ValueError, dict(page_table=torch.zeros(3, 0, dtype=torch.int32))), (ValueError, dict(cos=torch.ones(8, 16))),
    (ValueError, dict(cos=torch.ones(8, 32).double())), (ValueError, dict(sin=torch.ones(7, 32))), (ValueError, dict(cu_seqlens=_i(0, 3))),
    (TypeError, dict(cu_seqlens=torch.tensor([0, 1, 2, 3])))] + [(e, dict(pages=p)) for e, p in BAD_POOLS])
def test_append_refuses(error, more):
    with pytest.raises(error):
        _append(**more)


@pytest.mark.parametrize("error,more", [
    (ValueError, dict()), (ValueError, dict(q=_x(3, 3, 64))), (ValueError, dict(q=_x(3, 4, 96))), (ValueError, dict(q=_x(3, 17, 4, 64))),
    (ValueError, dict(q=_x(3, 0, 4, 64))), (ValueError, dict(q=_x(4, 64))), (TypeError, dict(q=_x(3, 4, 64).float())), (ValueError, dict(lengths=_i(1))),
    (ValueError, dict(scale=float("nan"))), (ValueError, dict(scale=float("inf"))),
    (ValueError, dict(page_table=torch.zeros(3, 2, 1, dtype=torch.int32)))] + [(e, dict(pages=p)) for e, p in BAD_POOLS])
def test_paged_attention_refuses(error, more):
    with pytest.raises(error):
        _attend(**more)


@pytest.mark.parametrize("error,more", [
    (ValueError, dict()), (ValueError, dict(q=_x(5, 3, 64))), (ValueError, dict(q=_x(5, 4, 80))), (ValueError, dict(k=_x(5, 2, 96))),
    (ValueError, dict(v=_x(5, 1, 64))), (ValueError, dict(k=_x(6, 2, 64), v=_x(6, 2, 64))), (TypeError, dict(v=_x(5, 2, 64).half())),
    (ValueError, dict(cu_seqlens_k=_i(0, 5))), (TypeError, dict(cu_seqlens=torch.tensor([0, 5]))), (ValueError, dict(cu_seqlens=_i())),
    (ValueError, dict(scale=float("inf"))), (ValueError, dict(q=_x(5, 0, 64)))])
def test_prompt_attention_refuses(error, more):
    with pytest.raises(error):
        _prompt(**more)


def test_c_entries_refuse_without_a_device(lib):
    assert lib.flashmhf_paged_append(None, None) == lib.flashmhf_paged_attention(None, None) == lib.flashmhf_prompt_attention(None, None) == -1
    assert lib.flashmhf_paged_attention_workspace_bytes(None) == 0

    def pages(**w):
        a = dict(k=4096, v=8192, k_scale=256, v_scale=512, page_stride=2 * 16 * 64, num_pages=3, n_kv=2, page_size=16, head_dim=64)
        a.update(w)
        return _lib.KVPagesParams(**a)

    def seq(**w):
        a = dict(lengths=1024, table=2048, table_stride=4, B=2, max_pages=4)
        a.update(w)
        return _lib.KVSequences(**a)

    def append(pages=pages(), seq=seq(), **w):
        a = dict(cu_seqlens=64, q=128, k=256, v=512, q_stride=(128, 64), k_stride=(128, 64), v_stride=(128, 64), q_out=1024, k_out=None,
                 cos_t=256, sin_t=512, tokens=5, n_q=2, max_positions=9)
        a.update(w)
        return lib.flashmhf_paged_append(C.byref(_lib.PagedAppendParams(pages=pages, seq=seq, **a)), None)

    def attend(pages=pages(), seq=seq(), **w):
        a = dict(q=128, o=256, q_stride=(128, 0, 64), o_stride=(128, 0, 64), lse=None, workspace=None, workspace_bytes=0, n_q=2, n_new=1, scale=0.1)
        a.update(w)
        return lib.flashmhf_paged_attention(C.byref(_lib.PagedAttentionParams(pages=pages, seq=seq, **a)), None)

    for call in (append, attend):
        for bad in (dict(head_dim=80), dict(page_size=48), dict(num_pages=0), dict(n_kv=0)):
            assert call(pages=pages(**bad)) == -2
        for bad in (dict(B=0), dict(max_pages=0), dict(max_pages=2**30, table_stride=2**31)):
            assert call(seq=seq(**bad)) == -2
        assert call(pages=pages(k=None)) == call(seq=seq(lengths=None)) == -1
        assert call(pages=pages(k=4100)) == call(seq=seq(table=2050)) == -5
        assert call(pages=pages(page_stride=2000)) == call(pages=pages(page_stride=1024)) == call(seq=seq(table_stride=3)) == -4
    assert append(tokens=0) == append(max_positions=0) == append(n_q=0) == append(cu_seqlens=None) == -2
    assert append(k=None) == append(q_out=None) == append(cos_t=None) == -1
    assert append(k=258) == append(k_out=8) == append(cu_seqlens=2) == -5
    assert append(v_stride=(100, 64)) == append(q_stride=(-8, 64)) == -4
    assert attend(n_q=3) == attend(n_new=0) == attend(n_new=17) == attend(scale=float("nan")) == -2
    assert attend(q=None) == -1 and attend(o=264) == -5 and attend(o_stride=(128, 0, 4)) == -4

    def prompt(**w):
        a = dict(q=128, k=256, v=512, o=1024, q_stride=(128, 64), k_stride=(128, 64), v_stride=(128, 64), o_stride=(128, 64), lse=None, cu_q=64,
                 cu_k=64, B=1, tokens_q=3, tokens_k=3, n_q=2, n_kv=2, head_dim=64, causal=1, scale=0.1)
        a.update(w)
        return lib.flashmhf_prompt_attention(C.byref(_lib.PromptAttentionParams(**a)), None)

    assert prompt(head_dim=65) == prompt(B=0) == prompt(tokens_q=0) == prompt(tokens_k=-1) == prompt(n_q=3) == prompt(scale=float("inf")) == -2
    assert prompt(q=None) == prompt(cu_k=None) == -1 and prompt(v=520) == prompt(lse=2) == -5 and prompt(k_stride=(128, 4)) == -4


def test_serving_struct_layouts():
    assert C.sizeof(_lib.KVPagesParams) == 56 and C.sizeof(_lib.KVSequences) == 32
    assert C.sizeof(_lib.PagedAppendParams) == 56 + 32 + 4 * 8 + 6 * 8 + 4 * 8 + 16
    assert C.sizeof(_lib.PagedAttentionParams) == 56 + 32 + 2 * 8 + 6 * 8 + 3 * 8 + 16
    assert C.sizeof(_lib.PromptAttentionParams) == 4 * 8 + 8 * 8 + 3 * 8 + 32


def test_pool_values():
    """values(): code times scale."""
    pages = _pages()
    pages.k.copy_(torch.tensor(3.5).to(torch.float8_e4m3fn))
    pages.k_scale.fill_(0.25)
    assert torch.equal(pages.values()[0], torch.full((4, 2, 16, 64), 0.875, dtype=torch.bfloat16))
