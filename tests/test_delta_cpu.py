"""Refusals of the gated delta rule and of dropout that need no device: the C ABI's argument checks and the operators' own."""
import ctypes

import pytest
import torch


@pytest.fixture(scope='module')
def lib():
    from dism_b200 import _lib, build
    build.build()
    return _lib.load()


@pytest.fixture(scope='module')
def flash(lib):
    import dism_b200
    dism_b200.install_dropin()
    import flash_dism
    return flash_dism


def message(lib):
    return lib.dism_last_error().decode()


def test_delta_arguments(lib):
    p, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4100)  # never dereferenced: every call below is rejected first
    big = 1 << 40

    def forward(q=p, initial=None, cu=None, sequences=2, n=100, key_heads=2, heads=4, d=64, dv=64, final=None, saved=p, size=big):
        return lib.dism_delta_forward(q, p, p, p, p, 1, initial, cu, sequences, n, key_heads, heads, d, dv, 1., p, final, 0, saved, size, None)
    assert forward(q=None) == 1 and 'null' in message(lib)
    assert forward(sequences=0) == 1 and forward(n=0) == 1 and 'positive' in message(lib)
    assert forward(n=2 ** 31 - 1) == 1
    assert forward(heads=5) == 1 and 'multiple' in message(lib)
    assert forward(heads=70000, key_heads=1) == 1 and '65535' in message(lib)
    assert forward(d=48) == 2 and 'unsupported' in message(lib)
    assert forward(dv=256) == 2 and 'unsupported' in message(lib)
    assert forward(q=odd) == 1 and '16-byte aligned' in message(lib)
    assert forward(initial=odd) == 1 and '16-byte aligned' in message(lib)
    assert forward(cu=ctypes.c_void_p(4098)) == 1
    assert forward(saved=None) == 1 and 'workspace' in message(lib)
    assert forward(size=1024) == 1 and 'workspace' in message(lib)
    assert forward(saved=ctypes.c_void_p(4224)) == 1 and 'misaligned' in message(lib)
    assert forward(sequences=2 ** 30, n=2 ** 20) == 1 and 'too many chunks' in message(lib)

    def backward(dout=p, d=64, saved=p, saved_size=big, work=p, size=big):
        return lib.dism_delta_backward(p, p, dout, None, 1, None, 2, 100, 2, 4, d, 64, 1., saved, saved_size, p, p, p, p, p, None, work, size, None)
    assert backward(dout=None) == 1 and 'null' in message(lib)
    assert backward(d=16) == 2
    assert backward(dout=odd) == 1 and 'aligned' in message(lib)
    assert backward(saved_size=64) == 1 and 'saved' in message(lib)
    assert backward(work=None) == 1 and 'workspace' in message(lib)
    assert backward(size=64) == 1 and 'workspace' in message(lib)

    def step(v=p, state=p, slots=p, pool=8, batch=4, heads=4, d=64):
        return lib.dism_delta_step(p, p, v, p, p, 0, state, slots, pool, batch, 2, heads, d, 64, 1., p, None)
    assert step(batch=0) == 1 and step(batch=70000) == 1 and step(pool=0) == 1
    assert step(slots=None, pool=3) == 1 and 'state of its own' in message(lib)
    assert step(state=None) == 1 and step(state=odd) == 1 and step(heads=3) == 1 and step(d=8) == 2
    assert lib.dism_delta_fault(None) == 1


def test_delta_sizes(lib):
    assert lib.dism_delta_saved(0, 2, 100, 4, 48, 64, 0, 0) == 0
    plain, kept = (lib.dism_delta_saved(0, 2, 100, 4, 64, 64, 0, backward) for backward in (0, 1))
    # two sequences of two chunks, four heads: table, T and P; for a backward the states and X besides
    assert plain >= 16 * (384 * 4 + 2 * 2560 * 2) and kept >= plain + 16 * (64 * 64 * 2 + 64 * 64 * 2)
    assert lib.dism_delta_saved(1, 3, 100, 4, 64, 64, 1, 1) > lib.dism_delta_saved(1, 3, 100, 4, 64, 64, 0, 1)
    assert lib.dism_delta_backward_workspace(0, 2, 100, 4, 64, 64) >= 16 * (64 * 64 * 2 + 64 * 4 * 4)


def test_dropout_arguments(lib):
    p = ctypes.c_void_p(4096)
    call = lambda kind=0, x=p, count=10, threshold=100, seed=p: lib.dism_dropout(kind, x, None, count, threshold, seed, 0, p, None)
    assert call(kind=3) == 2 and 'type' in message(lib)
    assert call(count=0) == 1 and call(count=(1 << 35) + 1) == 1
    assert call(threshold=-1) == 1 and call(threshold=65537) == 1 and 'threshold' in message(lib)
    assert call(x=None) == 1 and call(seed=None) == 1
    assert call(x=ctypes.c_void_p(4097)) == 1 and call(seed=ctypes.c_void_p(4100)) == 1 and 'aligned' in message(lib)


def test_operators_refuse_host_tensors(flash):
    q = torch.zeros(1, 4, 2, 32, dtype=torch.bfloat16)
    gates = torch.zeros(1, 4, 2)
    with pytest.raises(RuntimeError, match='invalid device'):
        flash.gated_delta_rule(q, q, q, gates, gates)
    with pytest.raises(RuntimeError, match='invalid device'):
        flash.gated_delta_step(q[:, 0], q[:, 0], q[:, 0], gates[:, 0], gates[:, 0], torch.zeros(1, 2, 32, 32))
    with pytest.raises(RuntimeError, match='invalid device'):
        flash.dropout_add(torch.zeros(4), None, .5, torch.zeros(2, dtype=torch.int64))
    for p in (-.1, 1.1, float('nan')):
        with pytest.raises(ValueError, match='probability'):
            flash.dropout_add(torch.zeros(4), None, p, torch.zeros(2, dtype=torch.int64))


def test_document_starts_are_validated_on_the_host(flash):
    from flash_dism import delta
    v = torch.zeros(1, 8, 2, 32)
    layout = flash.VarlenLayout.from_cu_seqlens(torch.tensor([0, 256], dtype=torch.int32), 256)
    with pytest.raises(ValueError, match='not both'):
        delta._documents(v, torch.tensor([0, 8], dtype=torch.int32), layout)
    with pytest.raises(ValueError, match='differ in length'):
        delta._documents(v, None, layout)
    for bad in ([0, 9], [1, 8], [0, 5, 4, 8], [0, -1, 8]):
        with pytest.raises(RuntimeError, match='invalid cu_seqlens'):
            delta._documents(v, torch.tensor(bad, dtype=torch.int32), None)
    with pytest.raises(RuntimeError, match='cu_seqlens must be int32'):
        delta._documents(v, torch.tensor([0, 8]), None)
    assert delta._documents(v, torch.tensor([0, 3, 3, 8], dtype=torch.int32), None).tolist() == [0, 3, 3, 8]


def test_host_starts_that_a_capture_uses_are_never_dropped(flash, monkeypatch):
    from flash_dism import delta
    upload = lambda starts: delta._host_starts(starts, torch.device('cpu'))
    first = upload([0, 11])
    monkeypatch.setattr(delta, '_capturing', lambda device: True, raising=False)
    assert upload([0, 11]) is first
    with pytest.raises(RuntimeError, match='inside a capture'):
        upload([0, 12])
    monkeypatch.setattr(delta, '_capturing', lambda device: False, raising=False)
    others = [upload([0, i]) for i in range(100, 200)]
    assert upload([0, 11]) is first and upload([0, 199]) is others[-1]
    assert len(delta._starts) <= 32


def test_philox_blocks():
    """The generator of the tests against the published known answers of Philox4x32-10: all zeros, all ones."""
    import numpy as np
    import delta_reference as reference
    first = reference.philox(8, 0, 0, 0).astype(np.uint32)
    words = [int(first[2 * i] | (first[2 * i + 1] << 16)) for i in range(4)]
    assert words == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]


def test_model_with_delta_layers_keeps_the_default_model():
    from dism_b200.model import DismLM, DeltaLayer, DismLayer
    with torch.device('meta'):
        plain, hybrid = DismLM(depth=2, width=64, heads=2, head_dim=32, vocab=64), DismLM(depth=2, width=64, heads=2, head_dim=32, vocab=64, delta_layers=(1,))
    assert [type(b.mixer) for b in plain.blocks] == [DismLayer] * 2 and [type(b.mixer) for b in hybrid.blocks] == [DismLayer, DeltaLayer]
    assert 'dropout_seed' not in dict(plain.named_buffers())
