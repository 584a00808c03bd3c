"""The TypeScript backend's hand-over of device memory, read as text (no Node here): tfjs-core's methods
are there and do what their executed Python twins do, in the same order."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _method(name):
    src = open(os.path.join(ROOT, "tfjs_b200", "ts", "src", "backend_cuda.ts")).read()
    m = re.search(r"^  (?:override |private )*%s\(.*?^  }$" % name, src, re.S | re.M)
    assert m, name
    return m.group(0)


def _in_order(text, *parts):
    at = -1
    for part in parts:
        at = text.find(part, at + 1)
        assert at >= 0, part


def test_the_methods_that_tfjs_core_calls():
    create = _method("createTensorFromGPUData")
    assert create.startswith("  override") and "this.fromForeign(" in create and "makeTensorFromTensorInfo" in create
    read = _method("readToGPU")
    assert read.startswith("  override")
    _in_order(read, "devicePtr(this.ctx, this.deviceIdForUpdate(", "exposed++", "shared = true", "signalStream",
              "holders", "this.incRef(dataId)", "makeTensorFromTensorInfo")
    update = _method("deviceIdForUpdate")
    _in_order(update, "this.launchReaders(", "this.deviceIdOf(", "host = undefined")


def test_memory_goes_behind_its_holders_work():
    _in_order(_method("freeBehind"), "binding.waitStream(", "binding.free(")
    drop = _method("drop")
    assert "this.freeBehind(" in drop
    assert "this.isExposed(" in _method("defer") and "this.disposeData(dataId)" in _method("defer")
