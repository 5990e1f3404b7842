from .dsalt_attention import DSALTAttention
from .dsalt_transformer import CounterDropout, DSALTTransformerBlock, SwiGLUFFN

__all__ = ["CounterDropout", "DSALTAttention", "DSALTTransformerBlock", "SwiGLUFFN"]
