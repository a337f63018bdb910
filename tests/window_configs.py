"""LFM2 layers with further attention options, registered under a name of their own."""
import contextlib

WINDOWED = "Lfm2OfWindowsForCausalLM"


@contextlib.contextmanager
def windowed_layers(window, **options):
    """For as long as this lasts, `WINDOWED` is an LFM2 whose attention sees `window` positions (None: all) and has these further options."""
    from dataclasses import dataclass

    from zig_ai_b200.config import register_architecture, unregister_architecture
    from zig_ai_b200.config.lfm2 import Lfm2Config
    from zig_ai_b200.models import lfm2

    @dataclass
    class Config(Lfm2Config):
        @classmethod
        def from_dict(cls, d):
            out = super().from_dict(d)
            out.architecture = WINDOWED
            return out

    def build(cfg):
        spec = lfm2.build_spec(cfg)
        spec.architecture = WINDOWED
        for layer in spec.layers:
            layer.block.params["mixer"].params.update(window=window, **options)
        return spec

    register_architecture(WINDOWED, Config, build)
    try:
        yield
    finally:
        unregister_architecture(WINDOWED)
