"""The Python wrappers of the paged-cache calls, without a GPU."""
import pytest
import torch


@pytest.mark.parametrize("code,kept", [(0, True), (601, False), (602, False), (603, False), (301, False)])
@pytest.mark.parametrize("clear", [True, False])
def test_workspaces_are_dropped_after_any_status(monkeypatch, code, kept, clear):
    """A 601 may hide behind an earlier code: the status word holds the first one."""
    from yllm_b200 import attn

    def call(name, st, clear_arg):
        assert name == "yattn_device_status" and clear_arg == int(clear)
        st._obj.value = code

    ws = {(0, 0, 128): torch.zeros(1)}
    monkeypatch.setattr(attn, "call", call)
    monkeypatch.setattr(attn, "_paged_ws", ws)
    assert attn.device_status(clear=clear) == code
    assert bool(ws) == kept


def test_strides_past_32_bits_are_refused():
    """The library takes strides as 32-bit numbers: one that does not fit would read other rows."""
    from yllm_b200 import attn
    meta = lambda stride, dt: torch.empty_strided((2, 256), (stride, 1), dtype=dt, device="meta")
    for stride, fits in ((256, True), (2 ** 32 - 8, True), (2 ** 32, False), (2 ** 32 + 256, False)):
        t, tables = meta(stride, torch.float16), meta(stride, torch.int32)
        dev = t.get_device()
        if fits:
            assert attn._token_stride(t, "q", 2, 256, torch.float16, dev) == stride
            assert attn._table_shape(tables, dev, 2) == (256, stride)
            continue
        with pytest.raises(ValueError, match="q must be"):
            attn._token_stride(t, "q", 2, 256, torch.float16, dev)
        with pytest.raises(ValueError, match="tables must be"):
            attn._table_shape(tables, dev, 2)
    one = torch.empty_strided((1, 256), (2 ** 40, 1), dtype=torch.float16, device="meta")   # a single row has no stride
    assert attn._token_stride(one, "q", 1, 256, torch.float16, one.get_device()) == 256


@pytest.mark.parametrize("max_new,given", [(-1, None), (0, 0), (3, 3), (2 ** 32, 2 ** 32 - 1), (2 ** 32 + 1, 2 ** 32 - 1)])
def test_max_new_reaches_the_library_as_it_is_meant(monkeypatch, max_new, given):
    """An upper bound that does not fit 32 bits stays an upper bound; a negative one is refused."""
    from yllm_b200 import attn
    seen = []
    monkeypatch.setattr(attn, "_act_of", lambda q: (1, q.dtype, q.get_device(), q.shape[0]))
    monkeypatch.setattr(attn, "_call_on", lambda name, dev, stream, *args: seen.append((name, args)))
    e = lambda *s, dt=torch.float16: torch.zeros(*s, dtype=dt)
    i32 = torch.int32
    args = (e(4, 256), e(4, 256), e(2, 16, 128), e(2, 16, 128), e(1, 3, dt=i32), e(2, dt=i32), e(1, dt=i32), max_new, 4, 2, 64)
    if given is None:
        with pytest.raises(ValueError, match="max_new"):
            attn.attn_paged(*args, workspace=e(16))
        return
    attn.attn_paged(*args, workspace=e(16))
    (name, passed), = seen
    names = ("out out_stride q q_stride gate gate_stride act kpool vpool n_pages page_size tables max_pages table_stride "
             "cu_new kv_len n_seqs n_tokens max_new n_heads n_kv_heads head_dim kv_dim workspace workspace_bytes").split()
    got = dict(zip(names, passed))
    assert name == "yattn_attn_paged" and len(passed) == len(names)
    assert (got["max_new"], got["n_tokens"], got["n_heads"], got["q_stride"]) == (given, 4, 4, 256)


def test_workspace_is_made_on_the_device_that_is_named(monkeypatch):
    """Device 0 is a device, not the default."""
    from yllm_b200 import attn
    made = []
    monkeypatch.setattr(attn, "_new_workspace", lambda head_dim, dev: made.append((head_dim, dev)))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 5)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    for device in (0, "cuda:0", torch.device("cuda", 0), 3, None, "cuda"):
        attn.paged_workspace(128, device)
    assert made == [(128, d) for d in (0, 0, 0, 3, 5, 5)]
    with pytest.raises(ValueError, match="CUDA"):
        attn.paged_workspace(128, "cpu")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_norm_weights_are_held_and_checked(monkeypatch, dtype):
    """The struct has bare pointers: the weights live as long as it does, and each call checks their size."""
    import gc
    import weakref

    from yllm_b200 import attn
    with pytest.raises(ValueError, match="q_w must be a CUDA"):
        attn.qk_norm(torch.ones(128, dtype=dtype), torch.ones(128, dtype=dtype), 1e-6)
    monkeypatch.setattr(attn, "_need", lambda t, dt, name: None)
    q_w, k_w = torch.ones(128, dtype=dtype), torch.ones(128, dtype=dtype)
    alive = weakref.ref(q_w)
    norm = attn.qk_norm(q_w, k_w, 1e-6)
    assert norm.q_w == q_w.data_ptr() and norm.k_w == k_w.data_ptr() and norm.w_f16 == (dtype == torch.float16)
    del q_w
    gc.collect()
    assert alive() is not None
    assert attn._norm_arg(None, 64) is None
    attn._norm_arg(norm, 128)
    attn._norm_arg(norm, 128, -1)
    with pytest.raises(ValueError, match="128 values for head_dim 256"):
        attn._norm_arg(norm, 256)
    with pytest.raises(ValueError, match="cuda:0"):
        attn._norm_arg(norm, 128, 0)
    attn._norm_arg(attn.YattnQkNorm(1, 2, 0, 1e-6), 256)      # a struct of the caller's own has pointers only
    norm = attn.qk_norm(torch.ones(64, dtype=dtype), torch.ones(32, dtype=dtype), 1e-6)
    with pytest.raises(ValueError, match="32 values"):
        attn._norm_arg(norm, 64)
