"""What tracing sees of the attention ops' outputs: the strides that the real ones have, whatever those of
the queries are (they allocate contiguous outputs)."""
import pytest
import torch

from tests.test_kv_cache import BF, fwd_args


def meta(**args):
    return {k: v.to("meta") if isinstance(v, torch.Tensor) else v for k, v in args.items()}


def queries():
    yield torch.empty(4, 5, 64, dtype=BF, device="meta").permute(1, 0, 2)             # [T, H, D] from [H, T, D]
    yield torch.empty(2, 4, 3, 64, dtype=BF, device="meta").permute(0, 2, 1, 3)       # [B, S, H, D] from [B, H, S, D]
    yield torch.empty(5, 9, 64, dtype=BF, device="meta")[:, :4]                       # a slice of a projection


@pytest.mark.parametrize("q", queries(), ids=["heads outside", "batched, heads outside", "slice"])
def test_strides_of_the_paged_form(q):
    from sgl_kernel import _ops  # noqa: F401

    a = meta(**fwd_args())
    a["q"] = q
    if q.dim() == 4:
        a["cu_seqlens_q"] = None
    names = ("k", "v", "k_descale", "v_descale", "page_table", "seqused_k", "cu_seqlens_q")
    rest = (*[a[n] for n in names], 3, None, True, -1, -1)
    outs = [torch.ops.sgl_kernel.fwd(**a)[:2], torch.ops.sgl_kernel.fwd_paged_fp8(q, *rest)]
    given = torch.empty_like(q)
    lse = torch.ops.sgl_kernel.fwd_paged_fp8_out(q, *rest, given)
    rows = (q.shape[0], q.shape[2], q.shape[1]) if q.dim() == 4 else (q.shape[1], q.shape[0])
    for out, s in outs:
        assert out.shape == q.shape and out.is_contiguous() and s.shape == rows and s.is_contiguous()
    assert lse.shape == rows and lse.is_contiguous()
    a["out"] = given                                                                  # a given one is returned
    out, s, *_ = torch.ops.sgl_kernel.fwd(**a)
    assert out.stride() == given.stride() and s.shape == rows


@pytest.mark.parametrize("q", list(queries())[1:], ids=["batched, heads outside", "slice"])
def test_strides_of_the_dense_form(q):
    from sgl_kernel import _ops  # noqa: F401

    if q.dim() == 3:
        q = q.unsqueeze(0)
    a = dict(fwd_args(), q=q, k=q, v=q, cu_seqlens_q=None, seqused_k=None, page_table=None, k_descale=None, v_descale=None,
             is_causal=False, max_seqlen_q=None)
    assert torch.ops.sgl_kernel.fwd(**a)[0].is_contiguous()
