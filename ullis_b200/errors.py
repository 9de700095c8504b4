"""Status codes of the C ABI (include/ullis_cuda.h) and the exception that carries them."""

OK, ERR_SHAPE, ERR_CHECKPOINT, ERR_CUDA, ERR_DEVICE_CHECK, ERR_NCCL, ERR_TIMEOUT, ERR_ARG, ERR_TOKEN, ERR_NOMEM = range(10)


class UllisCudaError(RuntimeError):
    def __init__(self, code: int, message: str):
        super().__init__(f"[ullis-cuda {code}] {message}")
        self.code = code
        self.message = message
