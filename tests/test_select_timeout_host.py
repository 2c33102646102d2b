"""CPU checks of the selection's timeout self-test entry: refused as starkv_select_pages is."""


def test_refusals():
    from starkv_b200 import _lib
    f = _lib.lib().starkv_selftest_select_timeout
    assert f(None, None, 0, None) == 22
    sizes = dict(dtype=1, n=2, num_heads=8, num_kv_heads=2, head_dim=128, num_blocks=9, block_size=16, max_blocks=4,
                 max_seq_len=1000, top=3, sinks=1, recent=1)

    def call(**change):
        a = _lib.SelectPagesArgs()
        for name, x in (sizes | change).items():
            setattr(a, name, x)
        return f(bytes(a), None, 0, None)
    assert call(n=0) == 0
    assert call(top=0) == call(sinks=3) == call(head_dim=96) == call() == 22
    assert call(dtype=2) == 101
