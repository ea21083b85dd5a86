"""The block-scaled KV cache's refusals: the C entry points check their
arguments before any launch, the Python calls their tensors; no GPU needed."""
import ctypes as C

import pytest
import torch

from torch2riscv_accelerator_b200 import _lib, ops

OK, EINVAL, EALIGN, ESCRATCH = _lib.W8A8_OK, _lib.W8A8_EINVAL, _lib.W8A8_EALIGN, _lib.W8A8_ESCRATCH


def blocks(**kw):
    a = dict(k=1 << 20, v=2 << 20, k_scale=3 << 20, v_scale=4 << 20, slots=2, kv_heads=2, capacity=128, head_dim=64,
             block=64, slot_stride=2 * 128 * 64, scale_stride=4)
    a.update(kw)
    return C.byref(_lib.W8A8KvBlocks(**a))


BAD_CACHES = [(dict(k=None), EINVAL), (dict(v_scale=None), EINVAL), (dict(slots=0), EINVAL),
              (dict(slots=65536), EINVAL), (dict(kv_heads=0), EINVAL), (dict(head_dim=272), EINVAL),
              (dict(head_dim=0), EINVAL), (dict(head_dim=40), EALIGN), (dict(block=48), EINVAL),
              (dict(block=8), EINVAL), (dict(capacity=96), EINVAL), (dict(capacity=0), EINVAL),
              (dict(k=(1 << 20) + 8), EALIGN), (dict(slot_stride=2 * 128 * 64 + 8), EALIGN),
              (dict(slot_stride=128 * 64), EINVAL), (dict(scale_stride=2), EINVAL), (dict(k_scale=2), EALIGN)]


@pytest.mark.parametrize("kw,status", BAD_CACHES)
def test_every_call_checks_the_cache(lib, kw, status):
    c = blocks(**kw)
    assert lib.w8a8_kvb_append(c, 16, 128, 16, 128, 0, 2, 16, None, None) == status
    assert lib.w8a8_kvb_read(c, 2, 16, None, 16, 16, 0, None) == status
    assert lib.w8a8_kvb_attn(c, 16, 256, 0, 4, 2, 16, None, 1.0, 16, None, 16, 1 << 30, None) == status
    assert lib.w8a8_kvb_evict(c, 16, 16, 4, 0, 0, None, None, 16, 32, None) == status
    assert lib.w8a8_kvb_attn_scratch_bytes(c, 4, 2, 1, 0, 0) == 0
    good = blocks(k=5 << 20, v=6 << 20, k_scale=7 << 20, v_scale=8 << 20)
    assert lib.w8a8_kvb_evict(good, 16, 16, 4, 0, 0, c, 64, 16, 32, None) == status


def test_append_and_read_arguments(lib):
    c = blocks()

    def append(k=16, ks=128, v=16, vs=128, t=0, rows=2, pos=16, start=None):
        return lib.w8a8_kvb_append(c, k, ks, v, vs, t, rows, pos, start, None)
    assert append(t=3) == EINVAL and append(k=None) == EINVAL and append(pos=None) == EINVAL
    assert append(rows=3) == EINVAL                                # one row per slot without offsets
    assert append(rows=-1, start=16) == EINVAL
    assert append(ks=127) == EINVAL and append(vs=64) == EINVAL    # rows overlap
    assert append(k=24) == EALIGN and append(ks=130) == EALIGN     # off the 16-byte grid
    assert append(ks=132, t=1) == EALIGN                           # 16-bit rows: multiples of 8 elements
    assert append(rows=0, start=16, k=None, v=None) == OK          # nothing to do, nothing launched
    assert lib.w8a8_kvb_read(c, 2, 16, None, 16, None, 0, None) == EINVAL
    assert lib.w8a8_kvb_read(c, 2, 16, None, 16, 8, 0, None) == EALIGN
    assert lib.w8a8_kvb_read(c, 2, 16, None, 16, 16, 7, None) == EINVAL
    assert lib.w8a8_kvb_read(c, 0, 16, 16, None, None, 0, None) == OK


def test_attention_arguments(lib):
    c = blocks()

    def attn(q=16, qs=256, t=0, heads=4, rows=2, pos=16, start=None, scale=1.0, out=16, mass=None, scratch=16,
             size=1 << 30):
        return lib.w8a8_kvb_attn(c, q, qs, t, heads, rows, pos, start, scale, out, mass, scratch, size, None)
    assert attn(heads=3) == EINVAL and attn(heads=0) == EINVAL     # a multiple of the KV heads
    assert attn(t=-1) == EINVAL and attn(q=None) == EINVAL and attn(out=None) == EINVAL
    assert attn(rows=1) == EINVAL and attn(pos=None) == EINVAL
    assert attn(qs=255) == EINVAL and attn(q=20) == EALIGN and attn(out=8) == EALIGN
    assert attn(mass=4) == EALIGN and attn(scratch=8, mass=16) == EALIGN
    assert attn(scale=float("nan")) == EINVAL and attn(scale=float("inf")) == EINVAL
    assert attn(rows=0, start=16, q=None, out=None) == OK
    need = lib.w8a8_kvb_attn_scratch_bytes(c, 4, 2, 1, 1, 0)
    assert need > 0 and attn(mass=16, size=need - 1) == ESCRATCH and attn(mass=16, scratch=None) == ESCRATCH


def test_evict_arguments(lib):
    c, d = blocks(), blocks(k=5 << 20, v=6 << 20, k_scale=7 << 20, v_scale=8 << 20)

    def evict(mass=16, count=16, keep=4, sink=0, recent=0, dst=None, dm=None, kept=16, out=32):
        return lib.w8a8_kvb_evict(c, mass, count, keep, sink, recent, dst, dm, kept, out, None)
    assert evict(keep=0) == EINVAL and evict(keep=129) == EINVAL
    assert evict(sink=3, recent=2) == EINVAL and evict(sink=-1) == EINVAL and evict(recent=-1) == EINVAL
    assert evict(sink=2 ** 31 - 1, recent=2 ** 31 - 1) == EINVAL
    assert evict(mass=None) == EINVAL and evict(kept=None) == EINVAL and evict(out=None) == EINVAL
    assert evict(out=16) == EINVAL                                 # the counts are read by every CTA
    assert evict(dst=d) == EINVAL and evict(dst=d, dm=16) == EINVAL
    assert evict(dst=c, dm=64) == EINVAL                           # overlapping source and destination
    assert evict(dst=blocks(k=5 << 20, v=6 << 20, k_scale=7 << 20, v_scale=8 << 20, slots=1), dm=64) == EINVAL
    assert evict(dst=blocks(k=5 << 20, v=6 << 20, k_scale=7 << 20, v_scale=8 << 20, block=32, scale_stride=8),
                 dm=64) == EINVAL


def test_python_calls_check_their_tensors():
    with pytest.raises(ValueError, match="block"):
        ops.kvb_cache(1, 1, 64, 64, block=40, device="cpu")
    c = ops.kvb_cache(2, 2, 100, 64, block=32, device="cpu")
    assert c.k.shape == (2, 2, 128, 64) and c.k_scale.shape == (2, 2, 4)
    pos = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kvb_attn(torch.zeros(2, 4, 64), c, pos)
    with pytest.raises(ValueError, match="int8"):
        ops.kvb_append(torch.zeros(2, 2, 64), torch.zeros(2, 2, 64), c._replace(k=c.k.float()), pos)
    with pytest.raises(ValueError, match="belong together"):
        ops.kvb_read(c._replace(v_scale=c.v_scale[:, :, :2]), pos, None, 2)
    with pytest.raises(ValueError, match="contiguous"):
        ops.kvb_read(c._replace(k=c.k.transpose(1, 2).contiguous().transpose(1, 2)), pos, None, 2)
    with pytest.raises(ValueError, match="start"):
        ops.kvb_attn_rows(torch.zeros(2, 4, 64), c, pos, None)


def test_torch_ops_have_fake_shapes():
    """torch.ops.w8a8.kvb_*: registered, what they write declared, shapes without a GPU."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    import torch2riscv_accelerator_b200.torch_ops as T
    assert {"kvb_append", "kvb_read", "kvb_attn", "kvb_attn_rows", "kvb_evict"} <= set(T.OPS)
    args = {a.name: a for a in torch.ops.w8a8.kvb_evict.default._schema.arguments}
    assert all(args[n].alias_info.is_write for n in ("k_codes", "k_scale", "v_codes", "v_scale", "mass"))
    with FakeTensorMode():
        c = (torch.empty(2, 3, 64, 32, dtype=torch.int8), torch.empty(2, 3, 2)) * 2
        i = torch.empty(2, dtype=torch.int32)
        q, mass = torch.empty(5, 6, 32, dtype=torch.bfloat16), torch.empty(2, 3, 64)
        k = torch.empty(5, 3, 32)
        s = torch.empty(3, dtype=torch.int32)
        assert torch.ops.w8a8.kvb_append(k, k, *c, i, s) is None
        assert torch.ops.w8a8.kvb_attn_rows(q, *c, i, s, mass).shape == q.shape
        assert torch.ops.w8a8.kvb_attn(q[:2], *c, i, None).dtype == torch.bfloat16
        assert [t.shape for t in torch.ops.w8a8.kvb_read(*c, i, s, 5)] == [(5, 3, 32)] * 2
        assert [t.shape for t in torch.ops.w8a8.kvb_evict(*c, mass, i, 7)] == [(2, 3, 7), (2,)]
