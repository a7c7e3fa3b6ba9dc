"""How finely the decode attention is split: the switch that sets it (CPU)."""


def test_the_split_target_is_asked_at_each_step(monkeypatch):
    """The switch may be set, changed and taken back while a program runs."""
    from fastgen_amd.kernels import ops

    monkeypatch.setattr(ops, "compute_units", lambda: 256)
    monkeypatch.delenv("FG_SPLIT_TARGET", raising=False)
    assert ops.attention_chunks_for(4, 8) == 36
    for target, chunks in (("512", 68), ("64", 12), ("0", 8), ("", 36)):
        monkeypatch.setenv("FG_SPLIT_TARGET", target)
        assert ops.attention_chunks_for(4, 8) == chunks
