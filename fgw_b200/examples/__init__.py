"""Small programs that run the framework's operators together."""
