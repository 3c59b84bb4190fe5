"""The package's own names: every call and constant of the 4-bit, rotary and dropout operators, next to the older ones."""


def test_names_of_the_package(built_lib):
    import kiln_b200
    from kiln_b200 import ops
    for name in ("quant4", "quant4_empty", "dequant4", "linear4", "linear4_dx", "padded_empty", "rope", "rope_freqs", "dropout", "Quant4", "MX4", "NV4", "EPI_GELU4",
                 "ROPE_HALF", "ROPE_INTERLEAVED", "ROPE_PLAIN", "ROPE_LINEAR", "ROPE_BASE", "ROPE_PARTS", "STATUS_RANGE", "linear16", "attn_self", "check_status"):
        assert getattr(kiln_b200, name) is getattr(ops, name), name
    assert not hasattr(kiln_b200, "quant5")
