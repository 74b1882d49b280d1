"""CPU: the paged-cache and rotary entry points refuse what they do not take before anything is launched, and the plain
64-bit statements that the GPU tests go by agree with dense attention and with torch's own sorting."""

import ctypes as C

import pytest
import torch

from kernels_b200 import _lib
from oracle import paged_oracle as PO

BAD, UNSUPPORTED, TOO_LARGE = 1, 2, 5


def _cache(**change):
    c = _lib.PagedCache()
    # (addresses that are never followed: every call below is refused or has nothing to do)
    c.k = c.v = c.page_table = c.lens = 4096
    c.B, c.H_kv, c.D, c.P, c.M, c.page, c.dtype = 2, 2, 64, 8, 4, 16, _lib.KB_F16
    for n, x in change.items():
        setattr(c, n, x)
    return c


CACHE_REFUSALS = [
    (dict(B=-1), BAD), (dict(H_kv=-1), BAD), (dict(P=-1), BAD), (dict(M=-1), BAD), (dict(page=0), BAD), (dict(dtype=4), UNSUPPORTED), (dict(dtype=-1), UNSUPPORTED),
    (dict(D=48), UNSUPPORTED), (dict(D=512), UNSUPPORTED), (dict(B=65536), TOO_LARGE), (dict(H_kv=65536), TOO_LARGE), (dict(M=1 << 16, page=1 << 15), TOO_LARGE),
    (dict(lens=None), BAD), (dict(page_table=None), BAD), (dict(k=None), BAD), (dict(v=None), BAD), (dict(dtype=3), BAD),
]


def _attention(**change):
    p = _lib.PagedAttentionParams()
    p.cache = change.pop("cache", _cache())
    p.q = p.o = p.workspace = 4096
    p.workspace_bytes, p.H, p.dtype, p.sm_scale = 1 << 40, 4, _lib.KB_F16, 1.0
    for n, x in change.items():
        setattr(p, n, x)
    return _lib.load().kb_paged_attention(C.byref(p), None)


def _write(**change):
    p = _lib.PagedWriteParams()
    p.cache = change.pop("cache", _cache())
    p.k.data = p.v.data = 4096
    p.T, p.dtype = 1, _lib.KB_F16
    for n, x in change.items():
        setattr(p, n, x)
    return _lib.load().kb_paged_write(C.byref(p), None)


def _evict(**change):
    p = _lib.PagedEvictParams()
    p.cache = change.pop("cache", _cache())
    p.weights = p.weights_out = p.row_positions = p.row_positions_out = p.lens_out = p.workspace = 4096
    p.workspace_bytes, p.budget, p.recent = 1 << 40, 8, 2
    for n, x in change.items():
        setattr(p, n, x)
    return _lib.load().kb_paged_evict(C.byref(p), None)


@pytest.mark.parametrize("call", [_attention, _write, _evict])
def test_cache_refusals(call):
    for change, status in CACHE_REFUSALS:
        assert call(cache=_cache(**change)) == status, change


def test_call_refusals():
    lib = _lib.load()
    for f in (lib.kb_paged_attention, lib.kb_paged_write, lib.kb_paged_evict, lib.kb_rotary):
        assert f(None, None) == BAD
    assert lib.kb_paged_attention_workspace_bytes(None) == 0 and lib.kb_paged_evict_workspace_bytes(None) == 0
    for change, status in [(dict(H=-4), BAD), (dict(H=3), BAD), (dict(context_size=-1), BAD), (dict(back_contexts=-1), BAD), (dict(q=None), BAD), (dict(o=None), BAD),
                           (dict(weights=4096), BAD), (dict(dtype=_lib.KB_BF16), UNSUPPORTED), (dict(dtype=3), UNSUPPORTED), (dict(H=65538), TOO_LARGE),
                           (dict(weights=4096, lse=4096, workspace=None), BAD), (dict(weights=4096, lse=4096, workspace_bytes=8), BAD),
                           (dict(weights=4096, lse=4096, workspace=4100), BAD), (dict(cache=_cache(H_kv=0)), BAD)]:
        assert _attention(**change) == status, change
    assert _attention(H=0) == 0 and _attention(cache=_cache(B=0)) == 0
    for change, status in [(dict(T=-1), BAD), (dict(dtype=_lib.KB_F32), UNSUPPORTED), (dict(dtype=3), UNSUPPORTED), (dict(T=1 << 30), TOO_LARGE)]:
        assert _write(**change) == status, change
    assert _write(T=0) == 0 and _write(cache=_cache(B=0)) == 0 and _write(cache=_cache(M=0)) == 0
    for change, status in [(dict(budget=0), BAD), (dict(recent=-1), BAD), (dict(lens_out=None), BAD), (dict(weights=None), BAD), (dict(row_positions_out=None), BAD),
                           (dict(weights_out=8192), BAD), (dict(row_positions_out=8192), BAD), (dict(lens_out=8192), BAD), (dict(workspace=None), BAD),
                           (dict(workspace_bytes=4), BAD), (dict(workspace=4097), BAD)]:
        assert _evict(**change) == status, change
    assert _evict(cache=_cache(B=0)) == 0
    r = _lib.RotaryParams()
    r.q.data = r.q_out = r.positions = r.inv_freq = 4096
    good = dict(B=1, H=1, T=1, D=64, R=32, axes=1, dtype=_lib.KB_F16)
    for change, status in [(dict(B=-1), BAD), (dict(H=-1), BAD), (dict(T=-1), BAD), (dict(D=65), UNSUPPORTED), (dict(dtype=3), UNSUPPORTED), (dict(R=0), BAD),
                           (dict(R=33), BAD),
                           (dict(axes=0), BAD), (dict(axes=9), BAD), (dict(axes=2), BAD), (dict(T=1 << 30, B=2), TOO_LARGE), (dict(q_out=None), BAD)]:
        for n, x in (good | dict(q_out=4096) | change).items():
            setattr(r, n, x)
        r.section_end[:] = [32] + [0] * 7
        assert lib.kb_rotary(C.byref(r), None) == status, change

def test_workspace_queries_refuse_what_the_calls_refuse():
    """The host-only queries are asked before the call: 0 for every block that the call does not take, head counts of which nothing can be shared out among them."""
    lib = _lib.load()

    def attention(**change):
        p = _lib.PagedAttentionParams()
        p.cache = change.pop("cache", _cache())
        p.q = p.o = p.lse = p.weights = 4096
        p.H, p.dtype, p.sm_scale = 4, _lib.KB_F16, 1.0
        p.q_stride[:] = [256, 64, 1]  # (dense heads: the tensor-core kernel's, where the head dim is)
        for n, x in change.items():
            setattr(p, n, x)
        return lib.kb_paged_attention_workspace_bytes(C.byref(p))

    def evict(**change):
        p = _lib.PagedEvictParams()
        p.cache = change.pop("cache", _cache())
        p.budget, p.recent = 8, 2
        for n, x in change.items():
            setattr(p, n, x)
        return lib.kb_paged_evict_workspace_bytes(C.byref(p))

    assert attention() > 0 and evict() > 0
    for change, _ in CACHE_REFUSALS:
        assert attention(cache=_cache(**change)) == 0 and evict(cache=_cache(**change)) == 0, change
    heads = _cache(H_kv=4)
    for change in (dict(H=-4), dict(H=3), dict(H=2, cache=heads), dict(H=1, cache=heads), dict(H=0), dict(H=65538), dict(context_size=-1), dict(back_contexts=-1),
                   dict(dtype=_lib.KB_BF16), dict(dtype=3), dict(dtype=-1), dict(cache=_cache(H_kv=0)), dict(cache=_cache(B=0)), dict(cache=_cache(B=40000), H=32768)):
        assert attention(**change) == 0, change
    for dtype in (_lib.KB_F32, _lib.KB_F16, _lib.KB_BF16):
        for H_kv in (2, 4, 64):
            for D in (16, 64, 128, 256):
                c = _cache(H_kv=H_kv, D=D, dtype=dtype)
                c.k_stride[:] = c.v_stride[:] = [16 * D * H_kv, 16 * D, D]
                for H in range(1, 3 * H_kv + 1):
                    assert (attention(H=H, dtype=dtype, cache=c) > 0) == (H % H_kv == 0), (dtype, H_kv, D, H)
    for change in (dict(budget=0), dict(budget=-1), dict(recent=-1), dict(cache=_cache(H_kv=0)), dict(cache=_cache(B=0))):
        assert evict(**change) == 0, change


@pytest.mark.parametrize("cls", [_lib.PagedCache, _lib.RotaryParams, _lib.PagedWriteParams, _lib.PagedAttentionParams, _lib.PagedEvictParams, _lib.SaBwdParams])
def test_packed_blocks_are_the_structures_bytes(cls):
    """Every number of a block, nested structures and arrays included, lands where the C structure has it."""
    def fill(x, numbers):
        for name, kind in x._fields_:
            if issubclass(kind, C.Structure):
                fill(getattr(x, name), numbers)
            elif issubclass(kind, C.Array):
                for i in range(kind._length_):
                    numbers.append(len(numbers) + 1)
                    getattr(x, name)[i] = numbers[-1]
            else:
                numbers.append(len(numbers) + 1)
                setattr(x, name, numbers[-1])
        return numbers

    block = cls()
    numbers = fill(block, [])
    packed = _lib.packer(cls)
    assert packed.size == C.sizeof(cls) and packed.pack(*numbers) == bytes(block)


def test_workspace_of_a_long_cache_passes_32_bits():
    lib = _lib.load()
    p = _lib.PagedAttentionParams()
    p.cache = _cache(B=64, M=1 << 14, page=64, H_kv=8, D=128)
    p.H, p.dtype, p.weights, p.lse = 64, _lib.KB_F16, 4096, 4096
    assert lib.kb_paged_attention_workspace_bytes(C.byref(p)) >= 64 * 64 * (1 << 20) * 4

def test_workspace_of_a_window_does_not_follow_the_table():
    """Scores take the room of the rows that a token can see."""
    lib = _lib.load()
    sizes = []
    for M in (1 << 6, 1 << 14):
        p = _lib.PagedAttentionParams()
        p.cache = _cache(B=64, M=M, page=64, H_kv=8, D=128)
        p.q_stride[:] = [32 * 128, 128, 1]
        p.H, p.dtype, p.weights, p.lse, p.context_size, p.back_contexts = 32, _lib.KB_F16, 4096, 4096, 512, 1
        sizes.append(lib.kb_paged_attention_workspace_bytes(C.byref(p)))
        p.weights = None
        sizes.append(lib.kb_paged_attention_workspace_bytes(C.byref(p)))
    assert sizes[0] == sizes[2] and sizes[0] - sizes[1] == sizes[2] - sizes[3] == 64 * 32 * 1024 * 4


def test_cpu_tensors_are_refused():
    from kernels_b200.streaming_attention import paged_attention, paged_cache_evict, paged_cache_write, rotary_embedding

    pages, table, lens = torch.zeros(4, 2, 16, 64), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    w, pos = torch.zeros(1, 2, 32), torch.zeros(1, 2, 32, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_attention(torch.zeros(1, 2, 64), pages, pages, table, lens)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_cache_write(torch.zeros(1, 2, 1, 64), torch.zeros(1, 2, 1, 64), pages, pages, table, lens)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_cache_evict(pages, pages, table, lens, w, pos, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        rotary_embedding(torch.zeros(1, 1, 1, 16), None, pos[0], torch.ones(8).double())


def test_attention_statement_agrees_with_the_whole_sequence_oracle():
    from oracle import streaming_attention_oracle as SO

    g = torch.Generator().manual_seed(0)
    T, c, back = 50, 8, 2
    q, k, v = (torch.randn(1, 2, T, 16, generator=g) for _ in range(3))
    table = torch.tensor([[3, 0, 5, 1, 6]], dtype=torch.int32)
    pages = [torch.zeros(7, 2, 10, 16) for _ in range(2)]
    PO.write(k, v, *pages, table, torch.tensor([T]))
    for n in (1, 8, 9, 33, 50):
        want = SO.streaming_attention_oracle(q, k, v, c, back, torch.tensor([n], dtype=torch.int32))[0]
        o = PO.attend(q[:, :, n - 1], *pages, table, torch.tensor([n]), c, back)[0]
        assert torch.allclose(o.float(), want[:, :, n - 1], atol=1e-5)


def test_eviction_statement_agrees_with_sorting():
    g = torch.Generator().manual_seed(1)
    n, budget, recent = 90, 40, 10
    pages = [torch.arange(8 * 16, dtype=torch.float32).view(8, 1, 16, 1).expand(8, 1, 16, 4).clone() for _ in range(2)]
    table, lens = torch.tensor([[4, 2, 7, 0, 1, 5]], dtype=torch.int32), torch.tensor([n], dtype=torch.int32)
    w, pos = torch.rand(1, 1, 96, generator=g), torch.arange(96, dtype=torch.int32).view(1, 1, 96).clone()
    rows = [pages[0][table[0, r // 16], 0, r % 16, 0].item() for r in range(n)]
    kept = set(range(n - recent, n)) | set(w[0, 0, : n - recent].topk(budget - recent).indices.tolist())
    PO.evict(*pages, table, lens, w, pos, budget, recent)
    assert lens.item() == budget and set(pos[0, 0, :budget].tolist()) == kept
    assert [pages[1][table[0, r // 16], 0, r % 16, 0].item() for r in range(budget)] == [rows[p] for p in pos[0, 0, :budget].tolist()]
    stay = [r for r in range(budget) if r in kept]
    assert all(pos[0, 0, r] == r for r in stay)
