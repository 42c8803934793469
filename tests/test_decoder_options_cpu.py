"""CPU: what a decoder's configuration becomes in the block driver's options. No kernel is launched."""
import pytest


def _options(**config):
    pytest.importorskip("torch")
    from ml_dataflow_b200.decoder import Decoder, DecoderConfig

    cfg = DecoderConfig(n_layers=1, d=64, n_heads=2, n_kv_heads=1, head_dim=32, n_experts=4, top_k=2, ffn=32, vocab=64, **config)
    dec = Decoder(cfg, 8, 8, device="cpu")
    return dec._options(dec.layers[0], dec.saved[0], dec.grads[0])


def test_sinks_without_a_window_are_no_option():
    """Without a window every key before a query is seen, the sinks among them: the op-by-op driver runs such a configuration, and the block
    driver, which refuses sinks without a window, must not be handed them."""
    assert _options(num_sinks=3) is None
    for config in (dict(qk_norm=True), dict(act8=True)):
        o = _options(num_sinks=3, **config)
        assert (o.window, o.num_sinks) == (0, 0), config
    o = _options(num_sinks=3, window=5)
    assert (o.window, o.num_sinks) == (5, 3)
