"""The counting proxy of the extension, over a stand-in for it."""

from types import SimpleNamespace

from representax_b200.ops._ext import _CountingModule


def test_calls_and_native_launches_are_counted_while_asked():
    native = [100]

    def fp4_ffn(launches):
        native[0] += launches

    module = _CountingModule(SimpleNamespace(kernel_launches=lambda: native[0], gemm=lambda: None,
                                             attention_backward=lambda: None, fp4_ffn=fp4_ffn, gated_ffn_apply=fp4_ffn))
    module.gemm()
    module.fp4_ffn(3)
    assert module.launches == 0 and not module.counting
    module.launches, module.counting = 0, True
    module.gemm()
    module.attention_backward()
    module.fp4_ffn(4)
    module.gated_ffn_apply(2)
    native[0] += 4  # a backward node, which no call of the proxy shows
    assert module.launches == 1 + 3 + 4 + 2 + 4
    module.counting = False
    module.fp4_ffn(3)
    module.gemm()
    assert module.launches == 14
    module.counting = True
    module.fp4_ffn(3)
    module.launches = 0
    module.fp4_ffn(2)
    assert module.launches == 2
