"""Python entry points of the native kernels (lazy: importing the package does not load the extension)."""
import importlib

_MODULES = ("grouped_gemm", "linear_loss", "tensor_lists")


def __getattr__(name):
    if name.startswith("__"):
        raise AttributeError(name)
    if name in _MODULES:
        return importlib.import_module(f"{__name__}.{name}")
    for module in _MODULES:
        mod = importlib.import_module(f"{__name__}.{module}")
        if hasattr(mod, name):
            value = getattr(mod, name)
            if not name.startswith("_") and callable(value):
                globals()[name] = value        # found once: an import inside a function does not search again
            return value
    raise AttributeError(name)
