from .layer import FP8DynamicLinear, FP8RotateQuantFA, add_fa_quant

__all__ = ["FP8DynamicLinear", "FP8RotateQuantFA", "add_fa_quant"]
